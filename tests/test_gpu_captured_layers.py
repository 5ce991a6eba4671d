"""LinearGQ in HIP graphs: several graphs of one process, captured on the same stream, replayed in any order, side by side and with
eager calls between them."""
import numpy as np
import pytest
import torch

from gq_testlib import activations, to_dev
from popxl_addons import _gq_hip
from popxl_addons.layers.linear_gq import LinearGQ
from popxl_addons.ops.group_quantize_decompress import group_quantize_compress

pytestmark = pytest.mark.gpu

IN, OUT = 4096, 4096  # (wide enough that decode and mid batches divide the input features, through the workspace)


@pytest.fixture(scope="module")
def layers(hip, device):
    made = {}
    for dim in (0, -1):
        w = torch.from_numpy(np.random.default_rng(dim + 2).normal(0, IN ** -0.5, (IN, OUT)).astype(np.float16)).to(device)
        layer = LinearGQ(OUT, bias=False, group_size=64, dim=dim)
        layer.init_variables(IN, torch.float16, device)
        names = ("weight_compressed", "weight_decompression_scale", "weight_decompression_bias")
        for name, a in zip(names, group_quantize_compress(w, 64, dim=dim)):
            layer.variables[name].data.copy_(a)
        made[dim] = layer
    return made


def _captured(call):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    return graph, held


@pytest.mark.parametrize("dim,backward,rows", [(-1, False, (1, 5, 40)), (-1, True, (40, 17, 100)), (0, False, (40, 17, 100)), (0, True, (1, 5, 40))])
def test_graphs_of_different_batches(hip, device, layers, dim, backward, rows):
    """Each graph has the arrival counters to itself: the last captured (and largest) is replayed first, all of them on streams of
    their own at once, and eager calls run between replays; every result is that of an eager call."""
    layer = layers[dim]
    call = layer.grad if backward else layer.build
    lib = hip.load()
    sizes = [(m, IN, OUT, 64) for m in rows]
    need = [(lib.gq_gemm_workspace_bytes if (dim == 0) != backward else lib.gq_linear_kn_workspace_bytes)(*s) for s in sizes]
    assert all(need) and len(set(need)) > 1
    xs = [torch.empty((m, IN), dtype=torch.float16, device=device) for m in rows]
    graphs, buffers = [], []
    for x in xs:
        before = {id(ws) for _, ws in _gq_hip._captured_workspaces.values()}
        graphs.append(_captured(lambda: call(x)))
        buffers += [b for b in _gq_hip._captured_workspaces.values() if id(b[1]) not in before]
        assert len(buffers) == len(graphs)
    assert len({number for number, _ in buffers}) == len({ws.data_ptr() for _, ws in buffers}) == len(rows)
    assert not {ws.data_ptr() for _, ws in buffers} & {ws.data_ptr() for ws in _gq_hip._kn_workspaces.values()}
    streams = [torch.cuda.Stream(device=device) for _ in rows]
    for turn in range(4):
        for i, x in enumerate(xs):
            x.copy_(to_dev(activations(len(x), IN, 10 * turn + i), device))
        want = [call(x) for x in xs]
        junk = torch.full((1 << 22,), 0xff, dtype=torch.uint8, device=device)  # (what freed memory may hold)
        del junk
        torch.cuda.synchronize()
        if turn % 2 == 0:
            for graph, _ in graphs[::-1]:
                graph.replay()
        else:
            for stream, (graph, _) in zip(streams, graphs):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for m, (_, held), w in zip(rows, graphs, want):
            assert torch.equal(held, w), (turn, m)


def test_several_layers_in_one_graph(hip, device, layers):
    """One stream of one capture uses one buffer, whose counters every call leaves zero; a forked stream has its own."""
    layer = layers[-1]
    x = to_dev(activations(3, IN, 5), device)
    want = layer.build(layer.build(x)), layer.build(x[1:])
    side = torch.cuda.Stream(device=device)

    def call():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        y = layer.build(layer.build(x))
        with torch.cuda.stream(side):
            z = layer.build(x[1:])
        main.wait_stream(side)
        return y, z

    graph, held = _captured(call)
    for _ in range(3):
        layer.build(x)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
