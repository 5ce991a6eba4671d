"""The 8-bit key/value cache: what append stores (code by code), what is read back, and the attention that reads it."""
import numpy as np
import pytest
import torch

from operators_testlib import BLOCK, PlainCache, assert_within, attend
from popxl_addons.ops.kv_cache_gq import KVCacheGQ, kv_cache_append, kv_cache_attention, kv_cache_gather
from popxl_addons.ops.rotary_pos_embed import RotaryPosEmbed, rotary_pos_embed

pytestmark = pytest.mark.gpu


def _int32(device, *arrays):
    return [torch.tensor(np.asarray(a), dtype=torch.int32, device=device) for a in arrays]


def _normal(seed, *shape):
    return np.random.default_rng(seed).normal(0, 1, shape).astype(np.float16)


def _codes(cache):
    k = cache.k_codes.cpu().numpy().astype(np.int32) - 128
    v = cache.v_codes.cpu().numpy().astype(np.int32).transpose(0, 1, 3, 2) - 128
    return k, v, cache.k_scale.cpu().numpy(), cache.v_scale.cpu().numpy()


def _table(lengths, seed, spare=2, width=0):
    need = [-(-n // BLOCK) for n in lengths]
    ids = np.random.default_rng(seed).permutation(sum(need) + spare)
    table, at = np.zeros((len(lengths), max([1, width] + need)), np.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, len(ids)


@pytest.mark.parametrize("heads,dim", [(1, 16), (3, 64), (2, 80), (2, 128), (1, 256)])
def test_append_codes(hip, device, heads, dim):
    """Steps of every kind -- first tokens, single ones into a block, growing and shrinking values, prompts over several blocks,
    sequences that wait -- against the definition applied token by token: codes and scales bit for bit."""
    steps = [[3, 0, 64], [1, 1, 0], [1, 70, 1], [60, 1, 1], [1, 0, 130], [7, 5, 6], [8, 9, 63], [0, 1, 1]]
    final = np.sum(steps, 0)
    table, n_blocks = _table(final, dim)
    cache, plain = KVCacheGQ(n_blocks, heads, dim, device), PlainCache(n_blocks, heads, dim)
    cache.k_codes.fill_(7), cache.v_codes.fill_(9)  # what a block held before does not matter
    cache.k_scale.fill_(1e9), cache.v_scale.fill_(1e9)
    lengths = np.zeros(3, int)
    for i, step in enumerate(steps):
        lengths += step
        offsets = np.concatenate([[0], np.cumsum(step)])
        size = np.float16([1, 3, 0.01, 40, 1, 8, 1, 0.5][i])
        k, v = (_normal(100 * i + j, offsets[-1], heads, dim) * size for j in range(2))
        if i == 5:
            v[:] = 0
        kv_cache_append(cache, torch.from_numpy(k).to(device), torch.from_numpy(v).to(device), *_int32(device, offsets, lengths, table))
        plain.append(k, v, offsets, lengths, table)
        got = _codes(cache)
        for b, n in enumerate(lengths):
            for p in range(-(-n // BLOCK)):
                block, slots = table[b, p], min(BLOCK, n - p * BLOCK)
                for j in range(2):
                    assert np.array_equal(got[2 + j][block], plain.scale[j][block]), (i, b, p, "kv"[j], "scale")
                    assert np.array_equal(got[j][block][:, :slots], plain.codes[j][block][:, :slots]), (i, b, p, "kv"[j])
    # whole sequences read back: one rounding of code * scale
    offsets = np.concatenate([[0], np.cumsum(lengths)])
    k, v = kv_cache_gather(cache, *_int32(device, offsets, lengths, table), tokens=int(offsets[-1]))
    for j, t in enumerate((k, v)):
        want = np.concatenate([plain.values(j, b, n, table) for b, n in enumerate(lengths)])
        assert np.array_equal(t.cpu().numpy(), want.astype(np.float16))


def test_append_stays_within_one_scale(hip, device):
    """64 tokens one by one, each larger than the last: every value within a scale of what was stored."""
    dim, table = 64, [[0]]
    cache = KVCacheGQ(1, 1, dim, device)
    k = _normal(5, 64, 1, dim) * np.float16(1.11) ** np.arange(64, dtype=np.float16)[:, None, None]
    for t in range(64):
        part = torch.from_numpy(k[t:t + 1]).to(device)
        kv_cache_append(cache, part, part, *_int32(device, [0, 1], [t + 1], table))
    got, _, scale, _ = _codes(cache)
    assert np.abs(got[0, 0] * scale[0, 0].astype(np.float64) - k[:, 0]).max() <= scale[0, 0]
    assert scale[0, 0] <= 2 * np.abs(k).max() / 127


def test_append_with_rotary_is_append_of_the_turned(hip, device):
    for layout, rotary_dim, dim in (("interleaved", 64, 256), ("half", 80, 80), ("half", 32, 64), ("interleaved", 8, 16)):
        lengths, fresh = [150, 70, 1], [100, 3, 1]
        table, n_blocks = _table(lengths, 3)
        offsets = np.concatenate([[0], np.cumsum(fresh)])
        batch = _int32(device, offsets, lengths, table)
        wide = torch.from_numpy(_normal(7, 104, 4 * dim + 8)).to(device)
        k, v = (wide[:, 8 + 2 * i * dim:8 + 2 * (i + 1) * dim].unflatten(1, (2, dim)) for i in range(2))
        rotary = RotaryPosEmbed(rotary_dim, layout=layout, device=device)
        one, two = (KVCacheGQ(n_blocks, 2, dim, device) for _ in range(2))
        kv_cache_append(one, k, v, *batch, rotary=rotary)
        positions = np.concatenate([np.arange(n - f, n) for n, f in zip(lengths, fresh)])
        kv_cache_append(two, rotary_pos_embed(k, *_int32(device, positions), rotary), v.contiguous(), *batch)
        for a, b in zip(_codes(one), _codes(two)):
            assert np.array_equal(a, b), layout


def test_padding_and_missing_blocks(hip, device):
    """More rows than tokens, rows behind the last sequence, block numbers outside the cache, lengths beyond the table."""
    dim, heads = 64, 2
    k, v = _normal(1, 300, heads, dim), _normal(2, 300, heads, dim)
    offsets, lengths = [0, 10, 80, 90, 250], [4, 70, 10, 1000]
    table = [[0, -1], [99, 1], [2 ** 31 - 1, 0], [2, 3]]
    cache = KVCacheGQ(5, heads, dim, device)
    batch = _int32(device, offsets, lengths, table)
    kv_cache_append(cache, torch.from_numpy(k).to(device), torch.from_numpy(v).to(device), *batch)
    plain = PlainCache(5, heads, dim)
    plain.append(k, v, offsets, [4, 70, 10, 128], table)  # the table holds 128 tokens: rows 122 ... 249 are the last ones
    got = _codes(cache)
    assert np.array_equal(got[2], plain.scale[0]) and np.array_equal(got[3], plain.scale[1])
    for block, slots in ((0, 4), (1, 6), (2, 64), (3, 64)):
        for j in range(2):
            assert np.array_equal(got[j][block][:, :slots], plain.codes[j][block][:, :slots])
            assert (got[j][block][:, slots:] == 0).all()
    assert (got[0][4] == 0).all()
    marks = tuple(torch.full((300, heads, dim), 77.0, dtype=torch.float16, device=device) for _ in range(2))
    kv_cache_gather(cache, *batch, tokens=300, out=marks)
    stored = np.zeros(300, bool)
    stored[6:10], stored[74:80], stored[122:250] = True, True, True
    for t in marks:
        t = t.cpu().numpy()
        assert (t[~stored] == 77).all() and np.abs(t[stored]).max() < 10
    q = _normal(3, 300, 2 * heads, dim)
    out = torch.full((300, 2 * heads, dim), 55.0, dtype=torch.float16, device=device)
    kv_cache_attention(torch.from_numpy(q).to(device), cache, *batch, out=out)
    out = out.cpu().numpy()
    assert (out[250:] == 55).all()  # behind the last sequence
    assert (out[:6] == 0).all() and (out[80:90] == 0).all() and (out[90:122] == 0).all()  # nothing to attend to
    for b, (row, length) in enumerate([(6, 4), (10, 70), (None, 0), (122, 128)]):
        if row is None:
            continue
        there = np.array([0 <= table[b][p // BLOCK] < 5 for p in range(length)])
        safe = [[t if 0 <= t < 5 else 4 for t in r] for r in table]
        want, room = attend(q[row:offsets[b + 1]], plain.values(0, b, length, safe), plain.values(1, b, length, safe),
                            length - (offsets[b + 1] - row), dim ** -0.5, there)
        assert_within(out[row:offsets[b + 1]], want, room, str(b))


def test_values_that_are_not_finite_stay_in_their_block(hip, device):
    dim, table, lengths = 64, [[0, 1]], [70]
    for bad in (np.inf, -np.inf, np.nan):
        k, v = _normal(1, 70, 2, dim), _normal(2, 70, 2, dim)
        k[66, 0, 5] = v[67, 1, 9] = bad
        cache = KVCacheGQ(2, 2, dim, device)
        batch = _int32(device, [0, 70], lengths, table)
        kv_cache_append(cache, torch.from_numpy(k).to(device), torch.from_numpy(v).to(device), *batch)
        kk, vv = (t.cpu().numpy() for t in kv_cache_gather(cache, *batch, tokens=70))
        assert not np.isfinite(kk[64:, 0]).any() and np.isfinite(kk[64:, 1]).all() and np.isfinite(kk[:64]).all()
        assert not np.isfinite(vv[64:, 1]).any() and np.isfinite(vv[64:, 0]).all() and np.isfinite(vv[:64]).all()
        out = kv_cache_attention(torch.from_numpy(_normal(3, 70, 2, dim)).to(device), cache, *batch).cpu().numpy()
        assert np.isfinite(out[:64]).all() and not np.isfinite(out[64:]).any()


def _filled(device, lengths, heads, dim, seed, spare=2, width=0):
    """A cache whose sequences hold drawn codes, everything else the worst that can lie there."""
    rng = np.random.default_rng(seed)
    table, n_blocks = _table(lengths, seed, spare, width)
    plain = PlainCache(n_blocks, heads, dim)
    for j in range(2):
        plain.codes[j][:] = np.clip(np.rint(rng.normal(0, 40, plain.codes[j].shape)), -127, 127)
        plain.scale[j][:] = rng.uniform(0.005, 0.05, plain.scale[j].shape)
    used = np.zeros(n_blocks, bool)
    for b, n in enumerate(lengths):
        used[table[b, :-(-n // BLOCK)]] = True
        if n % BLOCK:
            for j in range(2):
                plain.codes[j][table[b, n // BLOCK], :, n % BLOCK:] = 127
    for j in range(2):
        plain.scale[j][~used] = np.nan
    cache = KVCacheGQ.from_tensors(*(torch.from_numpy(np.ascontiguousarray(t)).to(device) for t in (
        (plain.codes[0] + 128).astype(np.uint8), (plain.codes[1] + 128).astype(np.uint8).transpose(0, 1, 3, 2), *plain.scale)))
    return cache, plain, table


SHAPES = [  # lengths, new tokens, kv heads, group, dim
    ([1], [1], 1, 1, 16),
    ([63, 64, 65, 1], [1, 1, 1, 1], 2, 1, 64),
    ([500], [1], 3, 1, 256),
    ([777, 3, 129], [1, 1, 1], 2, 8, 128),
    ([200, 90], [1, 1], 1, 7, 80),
    ([300], [1], 2, 20, 96),
    ([1000, 0, 17], [2, 0, 1], 2, 3, 64),
    ([130, 64, 250], [9, 64, 17], 2, 4, 128),
    ([90, 33], [90, 33], 2, 1, 256),
    ([513], [200], 1, 5, 112),
    ([5, 40, 300, 64, 65], [5, 1, 100, 64, 2], 4, 2, 64),
    ([320], [300], 2, 1, 128),
]


@pytest.mark.parametrize("lengths,fresh,heads,group,dim", SHAPES)
def test_attention_against_64_bits(hip, device, lengths, fresh, heads, group, dim):
    cache, plain, table = _filled(device, lengths, heads, dim, dim + len(lengths))
    offsets = np.concatenate([[0], np.cumsum(fresh)])
    q = _normal(dim, offsets[-1], heads * group, dim)
    got = kv_cache_attention(torch.from_numpy(q).to(device), cache, *_int32(device, offsets, lengths, table)).cpu().numpy()
    for b, n in enumerate(lengths):
        rows = slice(offsets[b], offsets[b + 1])
        want, room = attend(q[rows], plain.values(0, b, n, table), plain.values(1, b, n, table), n - fresh[b], dim ** -0.5)
        assert_within(got[rows], want, room, f"sequence {b}")


@pytest.mark.parametrize("size,scale", [(30.0, None), (1000.0, None), (0.0, None), (1.0, 0.0), (1.0, -0.7), (1e-4, 1.0)])
def test_attention_of_sharp_and_flat_scores(hip, device, size, scale):
    lengths, dim = [260, 31], 64
    cache, plain, table = _filled(device, lengths, 2, dim, 11)
    q = (_normal(4, 40, 4, dim) * np.float16(size)).astype(np.float16)
    offsets = [0, 30, 40]
    got = kv_cache_attention(torch.from_numpy(q).to(device), cache, *_int32(device, offsets, lengths, table), scale=scale).cpu().numpy()
    for b, n in enumerate(lengths):
        rows = slice(offsets[b], offsets[b + 1])
        k, v = plain.values(0, b, n, table), plain.values(1, b, n, table)
        want, room = attend(q[rows], k, v, n - (offsets[b + 1] - offsets[b]), dim ** -0.5 if scale is None else scale)
        # (a negative scale turns the error of the scores' sums, not its size)
        if scale is not None and scale < 0:
            _, more = attend(q[rows], -k, v, n - (offsets[b + 1] - offsets[b]), -scale)
            room = np.maximum(room, more)
        assert_within(got[rows], want, room, f"sequence {b}")


@pytest.mark.parametrize("scale", [None, 0.0, -0.4, 3.0])
@pytest.mark.parametrize("lengths,fresh,heads,group,dim,width", [([600], [90], 1, 1, 64, 64), ([400, 90], [120, 90], 2, 2, 128, 40),
                                                                  ([257], [257], 1, 1, 256, 100), ([700], [33], 1, 4, 80, 12)])
def test_attention_of_many_rows(hip, device, lengths, fresh, heads, group, dim, width, scale):
    """Prompts whose few tiles are divided over the keys (a wide table), at scales that turn, flatten and sharpen the scores;
    value scales of neighbouring blocks that differ by a thousand, and blocks of zeros."""
    cache, plain, table = _filled(device, lengths, heads, dim, 7 * dim + len(lengths), width=width)
    for j, c in enumerate((cache.k_scale, cache.v_scale)):
        for b, n in enumerate(lengths):
            for p in range(n // BLOCK):
                plain.scale[j][table[b, p]] *= [1, 1e-3, 0, 3, 1e3][(p + j) % 5] if j else [1, 0, 2][p % 3]
        c.copy_(torch.from_numpy(plain.scale[j]).to(device))
    offsets = np.concatenate([[0], np.cumsum(fresh)])
    q = _normal(dim, offsets[-1], heads * group, dim)
    got = kv_cache_attention(torch.from_numpy(q).to(device), cache, *_int32(device, offsets, lengths, table), scale=scale).cpu().numpy()
    for b, n in enumerate(lengths):
        rows = slice(offsets[b], offsets[b + 1])
        k, v = plain.values(0, b, n, table), plain.values(1, b, n, table)
        want, room = attend(q[rows], k, v, n - fresh[b], dim ** -0.5 if scale is None else scale)
        if scale is not None and scale < 0:
            _, more = attend(q[rows], -k, v, n - fresh[b], -scale)
            room = np.maximum(room, more)
        assert_within(got[rows], want, room, f"sequence {b}")


def test_many_rows_beside_a_block_that_is_not_finite(hip, device):
    """Rows in front of a block whose scales are not finite are as if it were not there."""
    for bad in (np.inf, np.nan):
        lengths, dim = [200], 64
        cache, plain, table = _filled(device, lengths, 1, dim, 41)
        q = torch.from_numpy(_normal(2, 200, 1, dim)).to(device)
        batch = _int32(device, [0, 200], lengths, table)
        want = kv_cache_attention(q, cache, *batch).cpu().numpy()
        for scale in (cache.k_scale, cache.v_scale):
            before = scale.clone()
            scale[table[0, 2]] = bad
            got = kv_cache_attention(q, cache, *batch).cpu().numpy()
            assert np.array_equal(got[:128], want[:128]) and not np.isfinite(got[128:]).any(1).any()
            scale.copy_(before)


@pytest.mark.parametrize("fresh", [3, 100])
def test_queries_that_are_not_finite_stay_in_their_row(hip, device, fresh):
    lengths, dim = [150], 64
    cache, plain, table = _filled(device, lengths, 1, dim, 51)
    q = _normal(3, fresh, 2, dim)
    batch = _int32(device, [0, fresh], lengths, table)
    want = kv_cache_attention(torch.from_numpy(q).to(device), cache, *batch).cpu().numpy()
    q[0, 1, 5], q[2, 0, 63], q[1, 1, 0] = np.nan, np.inf, -np.inf
    got = kv_cache_attention(torch.from_numpy(q).to(device), cache, *batch).cpu().numpy()
    bad = np.zeros((fresh, 2), bool)
    bad[0, 1] = bad[2, 0] = bad[1, 1] = True
    assert np.array_equal(got[~bad], want[~bad]) and np.isnan(got[bad]).any(1).all()


def test_attention_strides_streams_and_repeats(hip, device):
    lengths, fresh, heads, group, dim = [700, 65, 130], [1, 3, 20], 2, 4, 64
    cache, plain, table = _filled(device, lengths, heads, dim, 21)
    offsets = np.concatenate([[0], np.cumsum(fresh)])
    batch = _int32(device, offsets, lengths, table)
    q = torch.from_numpy(_normal(8, 24, heads * group, dim)).to(device)
    want = kv_cache_attention(q, cache, *batch)
    wide = torch.zeros((24, 2 * heads * group, dim + 24), dtype=torch.float16, device=device)
    wide[:, ::2, 8:8 + dim] = q
    view = wide[:, ::2, 8:8 + dim]
    assert torch.equal(kv_cache_attention(view, cache, *batch), want)
    odd = wide[:, ::2, 3:3 + dim]  # rows off a 16-byte border are copied first
    odd.copy_(q)
    assert torch.equal(kv_cache_attention(odd, cache, *batch), want)
    by_head = torch.full((heads * group, 24, dim + 1), 9.0, dtype=torch.float16, device=device)
    out = by_head.transpose(0, 1)[..., 1:]
    assert kv_cache_attention(q, cache, *batch, out=out) is out
    assert torch.equal(out, want) and (by_head[..., 0] == 9).all()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=device) for _ in range(2)]
    results = []
    for _ in range(3):
        for stream in streams:  # two calls at once, each with a workspace of its own
            with torch.cuda.stream(stream):
                results.append(kv_cache_attention(q, cache, *batch))
    torch.cuda.synchronize()
    assert all(torch.equal(r, want) for r in results)


def test_attention_beyond_32_bits(hip, device):
    """Blocks that lie more than 2^32 bytes into the cache."""
    heads, dim, lengths = 16, 256, [100]
    n_blocks = (1 << 32) // (heads * BLOCK * dim) + 40
    shape = (n_blocks, heads)
    cache = KVCacheGQ.from_tensors(torch.empty((*shape, BLOCK, dim), dtype=torch.uint8, device=device),
                                   torch.empty((*shape, dim, BLOCK), dtype=torch.uint8, device=device),
                                   torch.empty(shape, dtype=torch.float32, device=device), torch.empty(shape, dtype=torch.float32, device=device))
    table = [[n_blocks - 1, n_blocks - 3]]
    batch = _int32(device, [0, 100], lengths, table)
    k, v, q = (_normal(i, 100, heads, dim) for i in range(3))
    kv_cache_append(cache, torch.from_numpy(k).to(device), torch.from_numpy(v).to(device), *batch)
    kk, vv = (t.cpu().numpy() for t in kv_cache_gather(cache, *batch, tokens=100))
    assert np.abs(kk.astype(np.float64) - k).max() < np.abs(k).max() / 127 and np.abs(vv.astype(np.float64) - v).max() < np.abs(v).max() / 127
    plain = PlainCache(2, heads, dim)
    plain.append(k, v, [0, 100], lengths, [[0, 1]])
    out = kv_cache_attention(torch.from_numpy(q[-3:]).to(device), cache, *_int32(device, [0, 3], lengths, table)).cpu().numpy()
    want, room = attend(q[-3:], plain.values(0, 0, 100, [[0, 1]]), plain.values(1, 0, 100, [[0, 1]]), 97, dim ** -0.5)
    assert_within(out, want, room)


def test_shared_prefix(hip, device):
    """Two sequences that read the same first block."""
    dim = 64
    cache, plain, _ = _filled(device, [64 * 3], 1, dim, 31, spare=0)
    table, lengths = [[0, 1], [0, 2]], [100, 70]
    q = _normal(9, 2, 4, dim)
    got = kv_cache_attention(torch.from_numpy(q).to(device), cache, *_int32(device, [0, 1, 2], lengths, table)).cpu().numpy()
    for b in range(2):
        want, room = attend(q[b:b + 1], plain.values(0, b, lengths[b], table), plain.values(1, b, lengths[b], table), lengths[b] - 1, dim ** -0.5)
        assert_within(got[b:b + 1], want, room)


def test_nothing_to_do(hip, device):
    cache = KVCacheGQ(0, 2, 64, device)
    none = torch.empty((0, 2, 64), dtype=torch.float16, device=device)
    batch = _int32(device, [0], [], np.zeros((0, 3)))
    kv_cache_append(cache, none, none, *batch)
    assert kv_cache_attention(none, cache, *batch).shape == (0, 2, 64)
    assert kv_cache_gather(cache, *batch, tokens=0)[0].shape == (0, 2, 64)
    # a table without columns and a cache without blocks: nothing is there
    q = torch.ones((3, 2, 64), dtype=torch.float16, device=device)
    for table in (np.zeros((2, 0)), [[5, 6], [7, -3]]):
        batch = _int32(device, [0, 1, 3], [9, 100], table)
        kv_cache_append(cache, q, q, *batch)
        assert (kv_cache_attention(q, cache, *batch) == 0).all()


@pytest.mark.parametrize("new", [1, 40])
def test_codes_under_a_scale_of_zero_are_zeros(hip, device, new):
    """Tokens under a scale of 0 have the value 0 whatever their codes (a cache made elsewhere), and keep it when later tokens of
    their block bring a scale."""
    dim, heads, before = 64, 2, 10
    rng = np.random.default_rng(3)
    codes = [torch.from_numpy(rng.integers(1, 256, shape).astype(np.uint8)).to(device) for shape in ((2, heads, BLOCK, dim), (2, heads, dim, BLOCK))]
    scale = torch.tensor([[0.0, 0.5], [0.25, 0.0]], dtype=torch.float32, device=device)
    cache = KVCacheGQ.from_tensors(*codes, scale.clone(), scale.flip(1).contiguous())
    table = [[0], [1]]
    batch = _int32(device, [0, before, 2 * before], [before, before], table)
    values = [t.clone() for t in kv_cache_gather(cache, *batch, tokens=2 * before)]
    for i, t in enumerate(values):
        assert (t[:before, i] == 0).all() and (t[before:, 1 - i] == 0).all() and (t[:before, 1 - i] != 0).any()
    k, v = (torch.from_numpy(_normal(j, 2 * new, heads, dim)).to(device) for j in (1, 2))
    kv_cache_append(cache, k, v, *_int32(device, [0, new, 2 * new], [before + new] * 2, table))
    after = kv_cache_gather(cache, *_int32(device, [0, before + new, 2 * (before + new)], [before + new] * 2, table), tokens=2 * (before + new))
    for i, (old, got, x) in enumerate(zip(values, after, (k, v))):
        for b in range(2):
            there = got[b * (before + new):][:before + new]
            assert torch.equal(there[:before], old[b * before:][:before]), (i, b)  # (values of +-4 at most: scales of 0.25 and 0.5 do not grow)
            assert (there[before:] - x[b * new:][:new]).abs().max() <= 0.5


MIXED = [[64] + [1] * 40, [1] * 8, [3, 64, 17, 0, 130] + [1] * 90, [20, 2] + [1] * 20]  # few tokens a sequence on average, not in every block


@pytest.mark.parametrize("heads,dim", [(2, 64), (1, 256)])
@pytest.mark.parametrize("fresh", MIXED, ids=len)
def test_append_codes_of_mixed_batches(hip, device, heads, dim, fresh):
    """Batches of few new tokens a sequence whose blocks get from one token to all 64: codes and scales bit for bit."""
    before = np.random.default_rng(len(fresh)).integers(0, 100, len(fresh))
    lengths = before + fresh
    table, n_blocks = _table(lengths, dim)
    cache, plain = KVCacheGQ(n_blocks, heads, dim, device), PlainCache(n_blocks, heads, dim)
    for i, (step, length) in enumerate(((before, before), (np.array(fresh), lengths))):
        offsets = np.concatenate([[0], np.cumsum(step)])
        k, v = (_normal(10 * i + j, offsets[-1], heads, dim) * np.float16([1, 3][i]) for j in range(2))
        kv_cache_append(cache, torch.from_numpy(k).to(device), torch.from_numpy(v).to(device), *_int32(device, offsets, length, table))
        plain.append(k, v, offsets, length, table)
    got = _codes(cache)
    for b, n in enumerate(lengths):
        for p in range(-(-n // BLOCK)):
            block, slots = table[b, p], min(BLOCK, n - p * BLOCK)
            for j in range(2):
                assert np.array_equal(got[2 + j][block], plain.scale[j][block]), (b, p, "kv"[j], "scale")
                assert np.array_equal(got[j][block][:, :slots], plain.codes[j][block][:, :slots]), (b, p, "kv"[j])


@pytest.mark.parametrize("layout,rotary_dim,dim", [("half", 256, 256), ("interleaved", 256, 256), ("half", 160, 256), ("interleaved", 200, 208),
                                                   ("half", 64, 64), ("interleaved", 8, 16)])
@pytest.mark.parametrize("fresh", MIXED, ids=len)
def test_append_with_rotary_of_mixed_batches(hip, device, layout, rotary_dim, dim, fresh):
    """The same with keys turned on the way, more pairs than a wave has lanes among them: the bits of turning them first."""
    lengths = np.random.default_rng(len(fresh)).integers(0, 100, len(fresh)) + fresh
    table, n_blocks = _table(lengths, 5)
    batch = _int32(device, np.concatenate([[0], np.cumsum(fresh)]), lengths, table)
    k, v = (torch.from_numpy(_normal(j, sum(fresh), 2, dim)).to(device) for j in range(2))
    rotary = RotaryPosEmbed(rotary_dim, layout=layout, device=device)
    one, two = (KVCacheGQ(n_blocks, 2, dim, device) for _ in range(2))
    positions = np.concatenate([np.arange(n - f, n) for n, f in zip(lengths, fresh)])
    kv_cache_append(one, k, v, *batch, rotary=rotary)
    kv_cache_append(two, rotary_pos_embed(k, *_int32(device, positions), rotary), v, *batch)
    for a, b in zip(_codes(one), _codes(two)):
        assert np.array_equal(a, b)


def test_offsets_that_do_not_ascend(hip, device):
    """What rows then hold is not said; they stay rows of the tensors, blocks stay blocks of the cache and parts stay parts of the
    workspace, also where the units of all sequences are more than 32 bits count."""
    heads, dim = 1, 16
    cache, plain, table = _filled(device, [100, 30], heads, dim, 61)
    good = _int32(device, [0, 1, 4], [100, 30], table)
    q = torch.from_numpy(_normal(5, 4, heads, dim)).to(device)
    want = kv_cache_attention(q, cache, *good)
    for offsets in ([4, 0, 4], [-5, 9, 2], [2 ** 31 - 1, -2 ** 31, 3], [3, 2, 1]):
        batch = _int32(device, offsets, [100, 30], table)
        kv_cache_append(KVCacheGQ(5, heads, dim, device), q, q, *batch)
        kv_cache_gather(cache, *batch, tokens=4)
        kv_cache_attention(q, cache, *batch)
    # 512 sequences that are each given all 16384 rows (1024 tiles) over 8192 blocks, 2^32 units, and one with few more
    rows, blocks, many = 16384, 8192, 512
    wide = torch.full((2 * many + 1, blocks), -1, dtype=torch.int32, device=device)  # (no block is there)
    q2 = torch.zeros((rows, heads, dim), dtype=torch.float16, device=device)
    for extra in (0, 7, 2000):
        offsets = [0, rows] * many + [0, 16 if extra else 0]
        lengths = [blocks * BLOCK] * 2 * many + [extra * BLOCK]
        assert kv_cache_attention(q2, cache, *_int32(device, offsets, lengths), wide).shape == q2.shape
    torch.cuda.synchronize()
    assert torch.equal(kv_cache_attention(q, cache, *good), want)


@pytest.mark.parametrize("old", [1e-45, 1e-42, 1e-38, 1e-36, 2.0 ** -126, 3e-31, 4.7e-10, 1e-3])
@pytest.mark.parametrize("new", [1, 40])
def test_growth_from_small_scales(hip, device, old, new):
    """The least power of two, however far below the new tokens the scale is (a cache made elsewhere), and zeros under it."""
    dim, before = 64, 7
    old = np.float32(old)
    for x in (_normal(5, new, 1, dim), np.zeros((new, 1, dim), np.float16)):
        codes = [torch.from_numpy(np.random.default_rng(j).integers(1, 256, (1, 1, *s)).astype(np.uint8)).to(device) for j, s in enumerate(((BLOCK, dim), (dim, BLOCK)))]
        cache = KVCacheGQ.from_tensors(*codes, *(torch.full((1, 1), float(old), dtype=torch.float32, device=device) for _ in range(2)))
        had = _codes(cache)
        part = torch.from_numpy(x).to(device)
        kv_cache_append(cache, part, part, *_int32(device, [0, new], [before + new], [[0]]))
        got, need = _codes(cache), np.abs(x).max().astype(np.float32) / np.float32(127)
        e = 0
        while np.ldexp(np.float64(old), e) < need:
            e += 1
        scale = np.float32(np.ldexp(np.float64(old), e))
        for j in range(2):
            assert got[2 + j][0, 0] == scale
            assert np.array_equal(got[j][0, 0, before:before + new], np.clip(np.rint(x[:, 0].astype(np.float32) / scale), -127, 127))
            assert np.array_equal(got[j][0, 0, :before], np.rint(had[j][0, 0, :before] * 2.0 ** -e))


@pytest.mark.parametrize("fresh", [1, 70])
@pytest.mark.parametrize("order", [(0.02, 1e-40, 0.03), (1e-42, 0.05, 1e-45), (1e-33, 1e-40, 1e-36), (3e-29, 0.02, 2e-38), (1e-11, 500.0, 1e-13)])
def test_attention_of_small_scales(hip, device, order, fresh):
    """Scales that no binary16 token brings (a cache made elsewhere): what lies under them is next to nothing, in every order."""
    lengths, dim = [64 * 4 + 10], 64
    cache, plain, table = _filled(device, lengths, 2, dim, 71)
    for j, c in enumerate((cache.k_scale, cache.v_scale)):
        for p in range(5):
            plain.scale[j][table[0, p]] = order[(p + j) % 3]
        c.copy_(torch.from_numpy(plain.scale[j]).to(device))
    q = _normal(dim, fresh, 4, dim)
    got = kv_cache_attention(torch.from_numpy(q).to(device), cache, *_int32(device, [0, fresh], lengths, table)).cpu().numpy()
    want, room = attend(q, plain.values(0, 0, lengths[0], table), plain.values(1, 0, lengths[0], table), lengths[0] - fresh, dim ** -0.5)
    assert_within(got, want, room)
