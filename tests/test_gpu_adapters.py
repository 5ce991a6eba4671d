"""Low-rank adapters: forward and gradients against 64 bits, the plan, and the layer that has them beside its 4-bit weight."""
import numpy as np
import pytest
import torch

from gq_testlib import activations, normal_weight, normalised_error, to_dev
from operators_testlib import HALF16, TINY16, adapt, adapt_grad, assert_within
from popxl_addons.layers.linear_gq import LinearGQ
from popxl_addons.ops.group_quantize_decompress import group_quantize_compress_numpy
from popxl_addons.ops.low_rank_adapters import AdapterPlan, LowRankAdapters, low_rank_adapters, low_rank_adapters_grad

pytestmark = pytest.mark.gpu


def _problem(rows, k, n, rank, count, seed, ids=None):
    rng = np.random.default_rng(seed)
    if ids is None:
        ids = rng.integers(-1, count + 1, rows)  # (-1 and `count` are no adapters)
    return dict(x=rng.normal(0, 1, (rows, k)).astype(np.float16), y=rng.normal(0, 1, (rows, n)).astype(np.float16),
                down=rng.normal(0, k ** -0.5, (count, rank, k)).astype(np.float16), up=rng.normal(0, 0.3, (count, n, rank)).astype(np.float16),
                scaling=rng.uniform(-2, 2, count).astype(np.float32), ids=np.asarray(ids, np.int32))


def _on(device, p):
    d = {name: to_dev(a, device) for name, a in p.items()}
    return d, LowRankAdapters(d["down"], d["up"], d["scaling"]), AdapterPlan(d["ids"], len(p["down"]))


SIZES = [  # rows, in, out, rank, adapters
    (1, 64, 64, 16, 1),
    (3, 512, 640, 8, 2),
    (17, 1000, 1016, 13, 5),
    (40, 33, 70, 1, 3),
    (130, 264, 72, 64, 9),
    (65, 640, 136, 128, 2),
    (300, 128, 520, 40, 200),
    (1025, 520, 264, 32, 3),
    (1500, 96, 100, 24, 7),
    (1100, 136, 200, 100, 2),
    (2048, 64, 72, 5, 1),
    (1030, 264, 72, 64, 2),
    (4100, 72, 136, 100, 3),
    (8193, 72, 80, 16, 2),
    (8200, 40, 33, 20, 1),
]


@pytest.mark.parametrize("activation", [None, "relu", "gelu_tanh"])
@pytest.mark.parametrize("rows,k,n,rank,count", SIZES)
def test_forward(hip, device, rows, k, n, rank, count, activation):
    p = _problem(rows, k, n, rank, count, rows + k)
    d, adapters, plan = _on(device, p)
    want, room = adapt(p["x"], p["y"], p["down"], p["up"], p["scaling"], p["ids"], activation)
    apart = low_rank_adapters(d["x"], d["y"], adapters, plan, activation=activation)
    assert_within(apart.cpu().numpy(), want, room)
    assert np.array_equal(d["y"].cpu().numpy(), p["y"])
    assert low_rank_adapters(d["x"], d["y"], adapters, plan, activation=activation, out=d["y"]) is d["y"]
    assert torch.equal(apart, d["y"])


@pytest.mark.parametrize("rows,k,n,rank,count", SIZES)
def test_gradients(hip, device, rows, k, n, rank, count):
    p = _problem(rows, k, n, rank, count, rows + n)
    d, adapters, plan = _on(device, p)
    rng = np.random.default_rng(rank)
    dy = (rng.normal(0, 1e-3, (rows, n)) * 10.0 ** rng.integers(-2, 2, (rows, 1))).astype(np.float16)
    dx = rng.normal(0, 1e-3, (rows, k)).astype(np.float16)
    got = low_rank_adapters_grad(d["x"], to_dev(dy, device), adapters, plan, dx=to_dev(dx, device))
    want, rooms = adapt_grad(p["x"], dy, dx, p["down"], p["up"], p["scaling"], p["ids"])
    for name, g, w, room in zip(("dx", "d_down", "d_up"), got, want, rooms):
        assert_within(g.cpu().numpy(), w, room, name)
    again = low_rank_adapters_grad(d["x"], to_dev(dy, device), adapters, plan, dx=to_dev(dx, device))
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    alone = low_rank_adapters_grad(d["x"], to_dev(dy, device), adapters, plan)
    assert_within(alone[0].cpu().numpy(), *(lambda w, r: (w[0], r[0]))(*adapt_grad(p["x"], dy, 0 * dx, p["down"], p["up"], p["scaling"], p["ids"])))


@pytest.mark.parametrize("rows", [9, 1100])
def test_gradients_against_differences(hip, device, rows):
    """out is linear in each of x, down and up: <dy, out(t + e) - out(t - e)> = <grad, 2 e> for steps of any size, to the
    roundings of out (binary16) and of the gradient."""
    p = _problem(rows, 72, 80, 16, 2, 50)
    d, adapters, plan = _on(device, p)
    rng = np.random.default_rng(51)
    dy = rng.normal(0, 1, p["y"].shape).astype(np.float16)
    grads = low_rank_adapters_grad(d["x"], to_dev(dy, device), adapters, plan)
    for name, grad in zip(("x", "down", "up"), grads):
        e = rng.normal(0, 1, p[name].shape).astype(np.float16) * np.float16(np.abs(p[name]).max())
        sides, outs = (p[name] + e, p[name] - e), []
        for side in sides:
            t = dict(d, **{name: to_dev(side, device)})
            outs.append(low_rank_adapters(t["x"], None, LowRankAdapters(t["down"], t["up"], t["scaling"]), plan).cpu().numpy().astype(np.float64))
        step = sides[0].astype(np.float64) - sides[1].astype(np.float64)
        grad = grad.cpu().numpy().astype(np.float64)
        room = (np.abs(dy) * ((HALF16 + 2.0 ** -13) * (np.abs(outs[0]) + np.abs(outs[1])) + 2 * TINY16)).sum()
        room += (np.abs(step) * ((HALF16 if name == "x" else 2.0 ** -15) * np.abs(grad) + TINY16)).sum()
        assert abs((dy * (outs[0] - outs[1])).sum() - (grad * step).sum()) <= room, name


@pytest.mark.parametrize("ids", [[0] * 40, [-1] * 40, [5] * 39 + [2], list(range(40)), [7, -9, 2 ** 31 - 1, 6, 40, 39, -2 ** 31, 0] * 5])
def test_ids(hip, device, ids):
    p = _problem(40, 72, 88, 8, 40, 60, ids)
    d, adapters, plan = _on(device, p)
    want, room = adapt(p["x"], p["y"], p["down"], p["up"], p["scaling"], p["ids"])
    got = low_rank_adapters(d["x"], d["y"], adapters, plan).cpu().numpy()
    assert_within(got, want, room)
    without = (p["ids"] < 0) | (p["ids"] >= 40)
    assert np.array_equal(got[without], p["y"][without])
    dx, d_down, d_up = low_rank_adapters_grad(d["x"], d["y"], adapters, plan)
    unused = np.setdiff1d(np.arange(40), p["ids"])
    assert (dx.cpu().numpy()[without] == 0).all()
    assert (d_down.cpu().numpy()[unused] == 0).all() and (d_up.cpu().numpy()[unused] == 0).all()


def test_most_adapters(hip, device):
    """2048 adapters (three kinds of rows a thread of the plan), more rows than one pass of a wave."""
    p = _problem(5000, 24, 40, 2, 2048, 70)
    d, adapters, plan = _on(device, p)
    want, room = adapt(p["x"], p["y"], p["down"], p["up"], p["scaling"], p["ids"])
    assert_within(low_rank_adapters(d["x"], d["y"], adapters, plan).cpu().numpy(), want, room)
    dy = to_dev(p["y"], device)
    grads = low_rank_adapters_grad(d["x"], dy, adapters, plan)
    want, rooms = adapt_grad(p["x"], p["y"], 0 * p["x"], p["down"], p["up"], p["scaling"], p["ids"])
    for g, w, room in zip(grads, want, rooms):
        assert_within(g.cpu().numpy(), w, room)


def test_strided_rows_and_leading_axes(hip, device):
    p = _problem(24, 72, 88, 8, 4, 80)
    d, adapters, plan = _on(device, p)
    want = low_rank_adapters(d["x"], d["y"], adapters, plan)
    for pad, at in ((16, 8), (9, 5)):  # 16-byte aligned rows, and rows that are not
        wide = torch.full((24, 72 + 2 * pad), 5.0, dtype=torch.float16, device=device)
        out = torch.full((24, 88 + 2 * pad), 6.0, dtype=torch.float16, device=device)
        wide[:, at:at + 72], out[:, at:at + 88] = d["x"], d["y"]
        before = out.clone()
        view = out[:, at:at + 88]
        low_rank_adapters(wide[:, at:at + 72], view, adapters, plan, out=view)
        assert torch.equal(view, want)
        out[:, at:at + 88] = before[:, at:at + 88]
        assert torch.equal(out, before)
    folded = low_rank_adapters(d["x"].reshape(2, 3, 4, 72), d["y"].reshape(2, 3, 4, 88), adapters, plan)
    assert folded.shape == (2, 3, 4, 88) and torch.equal(folded.reshape(24, 88), want)


@pytest.mark.parametrize("size", [1e-4, 300.0])
def test_intermediate_range(hip, device, size):
    """x down^T far outside what binary16 holds well: it is kept in binary32 and scaled by a power of two."""
    p = _problem(20, 200, 64, 16, 2, 90)
    p["x"] = (p["x"] * np.float16(size)).astype(np.float16)
    p["down"] = (p["down"] * np.float16(20 if size > 1 else 0.05)).astype(np.float16)
    p["up"] = (p["up"] * np.float16(0.01 if size > 1 else 100)).astype(np.float16)
    p["y"] *= 0
    d, adapters, plan = _on(device, p)
    want, room = adapt(p["x"], p["y"], p["down"], p["up"], p["scaling"], p["ids"])
    assert_within(low_rank_adapters(d["x"], d["y"], adapters, plan).cpu().numpy(), want, room)


def test_values_that_are_not_finite_stay_in_their_rows(hip, device):
    p = _problem(40, 64, 64, 8, 3, 95)
    p["ids"][:] = np.arange(40) % 3
    p["x"][7, 3], p["x"][20, 0] = np.inf, np.nan
    p["down"][2, 1, 5] = np.inf  # the third adapter's rows
    d, adapters, plan = _on(device, p)
    got = low_rank_adapters(d["x"], d["y"], adapters, plan).cpu().numpy()
    bad = np.zeros(40, bool)
    bad[[7, 20]] = True
    bad[2::3] = True
    assert np.isfinite(got[~bad]).all() and not np.isfinite(got[bad]).all(1).any()


def test_update_of_a_plan_in_a_graph(hip, device):
    """A captured call follows new ids, x and y, and eager work between the replays does not disturb it."""
    p = _problem(33, 72, 88, 16, 6, 100)
    d, adapters, plan = _on(device, p)
    ids = d["ids"].clone()

    def step():
        plan.update(ids)
        return low_rank_adapters(d["x"], d["y"], adapters, plan, activation="relu"), low_rank_adapters_grad(d["x"], d["y"], adapters, plan)

    stream = torch.cuda.Stream(device=device)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    rng = np.random.default_rng(1)
    for _ in range(4):
        new = rng.integers(-1, 6, 33).astype(np.int32)
        ids.copy_(to_dev(new, device))
        d["x"].copy_(to_dev(rng.normal(0, 1, (33, 72)).astype(np.float16), device))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in (held[0], *held[1])]
        eager = AdapterPlan(to_dev(new, device), 6)
        want = [low_rank_adapters(d["x"], d["y"], adapters, eager, activation="relu"), *low_rank_adapters_grad(d["x"], d["y"], adapters, eager)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, want))


@pytest.mark.parametrize("dim", [0, -1])
@pytest.mark.parametrize("rows", [1, 5, 40, 200])
def test_layer_with_adapters(hip, device, oracle, dim, rows):
    """LinearGQ.build and grad beside the adapters: the layer's own result (to its tolerance) plus the adapters', and gradients."""
    k, n, rank, count = 256, 320, 16, 3
    w = normal_weight(n, k, 7)  # [out, in]
    packed, scale, bias = group_quantize_compress_numpy(w if dim == 0 else np.ascontiguousarray(w.T), 64)
    layer = LinearGQ(n, bias=True, group_size=64, dim=dim)
    layer.init_variables(k, torch.float16, device)
    out_bias = np.random.default_rng(1).normal(0, 1, n).astype(np.float16)
    names = ("weight_compressed", "weight_decompression_scale", "weight_decompression_bias", "bias")
    for name, value in zip(names, (packed, scale, bias, out_bias)):
        layer.variables[name].data.copy_(to_dev(value, device))
    weight = oracle.np_decompress(packed, scale, bias).astype(np.float64)
    weight = weight if dim == 0 else weight.T
    p = _problem(rows, k, n, rank, count, 3)
    d, adapters, plan = _on(device, p)
    y = layer.build(d["x"])
    got = layer.build(d["x"], adapters=adapters, plan=plan, activation="gelu_tanh")
    assert torch.equal(got, low_rank_adapters(d["x"], y, adapters, plan, activation="gelu_tanh"))
    base = p["x"].astype(np.float64) @ weight.T + out_bias
    want, _ = adapt(p["x"], base, p["down"], p["up"], p["scaling"], p["ids"], "gelu_tanh")
    assert normalised_error(got.cpu().numpy(), want) <= 1e-2
    dy = activations(rows, n, 8)
    dx = layer.grad(to_dev(dy, device))
    assert normalised_error(dx.cpu().numpy(), dy.astype(np.float64) @ weight) <= 1e-2
    full, d_down, d_up = layer.grad(to_dev(dy, device), d["x"], adapters, plan)
    want, rooms = adapt_grad(p["x"], dy, dx.cpu().numpy(), p["down"], p["up"], p["scaling"], p["ids"])
    for g, t, room in zip((full, d_down, d_up), want, rooms):
        assert_within(g.cpu().numpy(), t, room)


@pytest.mark.parametrize("count", [959, 960, 1019, 1023, 1024, 2048])
def test_plans_of_many_adapters(hip, device, count):
    """Counts of rows around the LDS that any launch may use."""
    p = _problem(300, 24, 40, 2, count, count)
    d, adapters, plan = _on(device, p)
    want, room = adapt(p["x"], p["y"], p["down"], p["up"], p["scaling"], p["ids"])
    assert_within(low_rank_adapters(d["x"], d["y"], adapters, plan).cpu().numpy(), want, room)


def test_calls_at_once(hip, device):
    """One plan and its adapters on two streams at once, forward and gradients, each call with a workspace of its own."""
    p = _problem(700, 520, 640, 24, 5, 90)
    d, adapters, plan = _on(device, p)
    want = low_rank_adapters(d["x"], d["y"], adapters, plan), *low_rank_adapters_grad(d["x"], d["y"], adapters, plan)
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream(device=device) for _ in range(2)], []
    for _ in range(4):
        for stream in streams:
            with torch.cuda.stream(stream):
                results.append((low_rank_adapters(d["x"], d["y"], adapters, plan), *low_rank_adapters_grad(d["x"], d["y"], adapters, plan)))
    torch.cuda.synchronize()
    for result in results:
        assert all(torch.equal(a, b) for a, b in zip(result, want))
