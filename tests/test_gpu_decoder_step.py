"""The operators together, as a decoder layer's attention uses them on its 4-bit projections: a fused q|k|v projection with adapters,
rotary positions, the 8-bit cache, attention over it, the output projection -- prompts, then decode steps, eager and captured."""
import numpy as np
import pytest
import torch

from gq_testlib import normalised_error, to_dev
from operators_testlib import PlainCache, adapt, assert_within, attend, rotate
from popxl_addons.layers.linear_gq import LinearGQ
from popxl_addons.ops.group_quantize_decompress import group_quantize_compress_numpy
from popxl_addons.ops.kv_cache_gq import KVCacheGQ, kv_cache_append, kv_cache_attention
from popxl_addons.ops.low_rank_adapters import AdapterPlan, LowRankAdapters
from popxl_addons.ops.rotary_pos_embed import RotaryPosEmbed, rotary_frequencies, rotary_pos_embed

pytestmark = pytest.mark.gpu

HIDDEN, Q_HEADS, KV_HEADS, DIM, ROTARY = 512, 8, 2, 64, 32
WIDTH = (Q_HEADS + 2 * KV_HEADS) * DIM


def _layer(rng, n_out, k_in, dim, device):
    w = rng.normal(0, k_in ** -0.5, (n_out, k_in)).astype(np.float16)
    arrays = group_quantize_compress_numpy(w if dim == 0 else np.ascontiguousarray(w.T), 64)
    layer = LinearGQ(n_out, bias=False, group_size=64, dim=dim)
    layer.init_variables(k_in, torch.float16, device)
    for name, a in zip(("weight_compressed", "weight_decompression_scale", "weight_decompression_bias"), arrays):
        layer.variables[name].data.copy_(to_dev(a, device))
    return layer, arrays


class Decoder:
    def __init__(self, device, dim, seed):
        rng = np.random.default_rng(seed)
        self.device, self.dim = device, dim
        self.qkv, self.qkv_arrays = _layer(rng, WIDTH, HIDDEN, dim, device)
        self.out, self.out_arrays = _layer(rng, HIDDEN, Q_HEADS * DIM, dim, device)
        self.down = rng.normal(0, HIDDEN ** -0.5, (3, 8, HIDDEN)).astype(np.float16)
        self.up = rng.normal(0, 0.2, (3, WIDTH, 8)).astype(np.float16)
        self.scaling = np.array([0.5, 1, 2], np.float32)
        self.adapters = LowRankAdapters(to_dev(self.down, device), to_dev(self.up, device), to_dev(self.scaling, device))
        self.rotary = RotaryPosEmbed(ROTARY, device=device)
        self.cache = KVCacheGQ(12, KV_HEADS, DIM, device)

    def step(self, x, positions, plan, offsets, seq_lens, table):
        """Every intermediate result, as the layer's forward pass makes them."""
        qkv = self.qkv.build(x, adapters=self.adapters, plan=plan)
        heads = qkv.unflatten(1, (Q_HEADS + 2 * KV_HEADS, DIM))
        q, k, v = heads.split((Q_HEADS, KV_HEADS, KV_HEADS), 1)
        turned = rotary_pos_embed(q, positions, self.rotary)
        kv_cache_append(self.cache, k, v, offsets, seq_lens, table, rotary=self.rotary)
        values = kv_cache_attention(turned, self.cache, offsets, seq_lens, table)
        return qkv, turned, values, self.out.build(values.flatten(1))


def _batch(device, ids, lengths, fresh, table):
    offsets = np.concatenate([[0], np.cumsum(fresh)])
    positions = np.concatenate([np.arange(n - f, n) for n, f in zip(lengths, fresh)])
    row_ids = np.repeat(ids, fresh)
    return [torch.tensor(np.asarray(a), dtype=torch.int32, device=device) for a in (positions, row_ids, offsets, lengths, table)]


@pytest.mark.parametrize("dim", [0, -1])
def test_prompts_and_decode_steps(hip, device, oracle, dim):
    """Each result against 64 bits on what the step before it gave (so that each tolerance is its own operator's)."""
    decoder, rng = Decoder(device, dim, 3), np.random.default_rng(5)
    weight = oracle.np_decompress(*decoder.qkv_arrays).astype(np.float64)
    out_weight = oracle.np_decompress(*decoder.out_arrays).astype(np.float64)
    if dim != 0:
        weight, out_weight = weight.T, out_weight.T
    table, ids, plain = [[7, 2, 9], [0, 11, 3], [4, 5, 1]], np.array([2, -1, 0]), PlainCache(12, KV_HEADS, DIM)
    lengths = np.zeros(3, int)
    for fresh in ([70, 1, 130], [1, 1, 1], [1, 1, 1], [3, 64, 0], [1, 1, 1]):
        lengths += fresh
        x = rng.normal(0, 1, (sum(fresh), HIDDEN)).astype(np.float16)
        positions, row_ids, offsets, seq_lens, blocks = _batch(device, ids, lengths, fresh, table)
        plan = AdapterPlan(row_ids, 3)
        qkv, turned, values, y = (t.cpu().numpy() for t in decoder.step(to_dev(x, device), positions, plan, offsets, seq_lens, blocks))
        want, _ = adapt(x, x.astype(np.float64) @ weight.T, decoder.down, decoder.up, decoder.scaling, row_ids.cpu().numpy())
        assert normalised_error(qkv, want) <= 1e-2
        heads = qkv.reshape(len(x), -1, DIM)
        p = positions.cpu().numpy()
        assert_within(turned, *rotate(heads[:, :Q_HEADS], p, *rotary_frequencies(ROTARY), "interleaved"), "q")
        k = rotary_pos_embed(to_dev(heads[:, Q_HEADS:Q_HEADS + KV_HEADS], device), positions, decoder.rotary).cpu().numpy()
        plain.append(k, heads[:, Q_HEADS + KV_HEADS:], offsets.cpu().numpy(), lengths, table)
        o = offsets.cpu().numpy()
        for b, n in enumerate(lengths):
            rows = slice(o[b], o[b + 1])
            want, room = attend(turned[rows], plain.values(0, b, n, table), plain.values(1, b, n, table), n - fresh[b], DIM ** -0.5)
            assert_within(values[rows], want, room, f"sequence {b}")
        assert normalised_error(y, values.reshape(len(x), -1).astype(np.float64) @ out_weight.T) <= 1e-2


@pytest.mark.parametrize("dim", [0, -1])
def test_captured_decode_step(hip, device, dim):
    """A decode step in a HIP graph: replays follow x, positions, ids and lengths that change in place, with eager work between
    them, and give the bits of the eager step."""
    eager, graphed = Decoder(device, dim, 8), Decoder(device, dim, 8)
    rng = np.random.default_rng(9)
    table = [[0, 1, 2], [3, 4, 5], [6, 7, 8], [9, 10, 11]]
    lengths = np.array([60, 1, 127, 64])
    x0 = to_dev(rng.normal(0, 1, (lengths.sum(), HIDDEN)).astype(np.float16), device)
    positions, row_ids, offsets, seq_lens, blocks = _batch(device, [0, 1, 2, -1], lengths, lengths, table)
    for d in (eager, graphed):
        d.step(x0, positions, AdapterPlan(row_ids, 3), offsets, seq_lens, blocks)
    x = torch.zeros((4, HIDDEN), dtype=torch.float16, device=device)
    positions, row_ids, offsets, seq_lens, blocks = _batch(device, [0, 1, 2, -1], lengths + 1, [1] * 4, table)
    plan = AdapterPlan(row_ids, 3)

    def step():
        plan.update(row_ids)
        return graphed.step(x, positions, plan, offsets, seq_lens, blocks)

    state = [t.clone() for t in (graphed.cache.k_codes, graphed.cache.v_codes, graphed.cache.k_scale, graphed.cache.v_scale)]
    stream = torch.cuda.Stream(device=device)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for mine, before in zip((graphed.cache.k_codes, graphed.cache.v_codes, graphed.cache.k_scale, graphed.cache.v_scale), state):
        mine.copy_(before)  # (the warm-up stored a token)
    for i in range(6):
        lengths += 1
        new_ids = rng.integers(-1, 3, 4)
        x.copy_(to_dev(rng.normal(0, 1 + i, (4, HIDDEN)).astype(np.float16), device))
        for mine, new in zip((positions, row_ids, seq_lens), (lengths - 1, new_ids, lengths)):
            mine.copy_(torch.tensor(new, dtype=torch.int32, device=device))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = eager.step(x, positions, AdapterPlan(row_ids, 3), offsets, seq_lens, blocks)
        torch.cuda.synchronize()
        for name, a, b in zip(("qkv", "q", "values", "y"), got, want):
            assert torch.equal(a, b), (i, name)
    for name in ("k_codes", "v_codes", "k_scale", "v_scale"):
        assert torch.equal(getattr(eager.cache, name), getattr(graphed.cache, name)), name


@pytest.mark.parametrize("dim", [0, -1])
def test_two_captured_steps(hip, device, dim):
    """Steps of two batches in graphs of their own, on one cache, the second captured replayed first and eager steps between them:
    the bits of eager steps."""
    eager, graphed = Decoder(device, dim, 18), Decoder(device, dim, 18)
    rng = np.random.default_rng(19)
    tables, lengths = [[[0, 1], [2, 3], [4, 5]], [[6, 7], [8, 9]]], [np.array([60, 3, 64]), np.array([63, 100])]
    state = []
    for table, n in zip(tables, lengths):
        x0 = to_dev(rng.normal(0, 1, (n.sum(), HIDDEN)).astype(np.float16), device)
        ids = list(range(len(n)))
        positions, row_ids, offsets, seq_lens, blocks = _batch(device, ids, n, n, table)
        for d in (eager, graphed):
            d.step(x0, positions, AdapterPlan(row_ids, 3), offsets, seq_lens, blocks)
        x = torch.zeros((len(n), HIDDEN), dtype=torch.float16, device=device)
        arrays = _batch(device, ids, n + 1, [1] * len(n), table)
        state.append((x, arrays, AdapterPlan(arrays[1], 3)))

    def step(decoder, i):
        x, (positions, row_ids, offsets, seq_lens, blocks), plan = state[i]
        plan.update(row_ids)
        return decoder.step(x, positions, plan, offsets, seq_lens, blocks)

    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step(graphed, i)
        graphs.append((graph, held))
    for turn in range(4):
        for i in (1, 0):
            lengths[i] += 1
            x, (positions, row_ids, _, seq_lens, _), _ = state[i]
            x.copy_(to_dev(rng.normal(0, 1 + turn, x.shape).astype(np.float16), device))
            for mine, new in zip((positions, row_ids, seq_lens), (lengths[i] - 1, rng.integers(-1, 3, len(x)), lengths[i])):
                mine.copy_(torch.tensor(new, dtype=torch.int32, device=device))
            want = step(eager, i)
            graphs[i][0].replay()
            torch.cuda.synchronize()
            for name, a, b in zip(("qkv", "q", "values", "y"), graphs[i][1], want):
                assert torch.equal(a, b), (turn, i, name)
