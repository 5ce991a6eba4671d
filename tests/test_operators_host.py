"""Operators beside the projections, as far as they need no GPU: refusals of the C entry points and of the Python calls, and the
frequencies of stretched contexts."""
import ctypes
import math
import sys

import numpy as np
import pytest
import torch

from launch_recorder import launches
from popxl_addons import _gq_hip
from popxl_addons._gq_hip import GQ_ERR_BAD_SHAPE, GQ_ERR_MISALIGNED, GQ_ERR_NULL_POINTER, GQ_ERR_UNSUPPORTED
from popxl_addons.layers.linear_gq import LinearGQ
from popxl_addons.ops.kv_cache_gq import KVCacheGQ, kv_cache_append, kv_cache_attention
from popxl_addons.ops.low_rank_adapters import AdapterPlan, LowRankAdapters, low_rank_adapters
from popxl_addons.ops.rotary_pos_embed import RotaryPosEmbed, rotary_frequencies, rotary_pos_embed


def _refused(code, name, *args):
    with pytest.raises(_gq_hip.GQHipError) as e:
        _gq_hip.call(name, *args)
    assert e.value.code == code, str(e.value)
    return str(e.value)


def _address(c):
    return ctypes.byref(c)


def test_rotary_refusals():
    ok = dict(t=16, t_token=64, t_head=32, positions=16, rotary=(16, 1.0, 32, 0), out=32, o_token=64, o_head=32, tokens=3, heads=2, dim=32)

    def refused(code, **change):
        a = {**ok, **change}
        rotary = a["rotary"] and _gq_hip.Rotary(*a["rotary"])
        return _refused(code, "gq_rotary_f16", a["t"], a["t_token"], a["t_head"], a["positions"], rotary and _address(rotary), 0, a["out"],
                        a["o_token"], a["o_head"], a["tokens"], a["heads"], a["dim"], None)

    refused(GQ_ERR_NULL_POINTER, rotary=None)
    refused(GQ_ERR_NULL_POINTER, t=0)
    refused(GQ_ERR_NULL_POINTER, positions=0)
    refused(GQ_ERR_NULL_POINTER, out=0)
    refused(GQ_ERR_NULL_POINTER, rotary=(0, 1.0, 32, 0))
    refused(GQ_ERR_MISALIGNED, t=17)
    refused(GQ_ERR_MISALIGNED, positions=18)
    refused(GQ_ERR_MISALIGNED, rotary=(20, 1.0, 32, 0))
    refused(GQ_ERR_BAD_SHAPE, tokens=-1)
    for rotary_dim in (0, -2, 31, 34):
        assert "rotary_dim" in refused(GQ_ERR_BAD_SHAPE, rotary=(16, 1.0, rotary_dim, 0))
    refused(GQ_ERR_UNSUPPORTED, rotary=(16, 1.0, 258, 0), dim=300)
    assert "layout" in refused(GQ_ERR_UNSUPPORTED, rotary=(16, 1.0, 32, 2))
    refused(GQ_ERR_UNSUPPORTED, t_head=-32)
    refused(GQ_ERR_UNSUPPORTED, o_token=(1 << 30) + 1)
    assert "in place" in refused(GQ_ERR_UNSUPPORTED, out=16, o_token=128)
    _gq_hip.call("gq_rotary_f16", 0, 0, 0, 0, _address(_gq_hip.Rotary(0, 1.0, 32, 0)), 0, 0, 0, 0, 0, 2, 32, None)  # no tokens


def test_kv_refusals():
    cache_ok, batch_ok = [16, 16, 16, 16, 10, 2, 64], [16, 16, 16, 3, 4, 5]

    def refused(code, name, cache=(), batch=(), **change):
        c, b = list(cache_ok), list(batch_ok)
        for i, value in cache:
            c[i] = value
        for i, value in batch:
            b[i] = value
        c, b = _gq_hip.KvCache(*c), _gq_hip.KvBatch(*b)
        a = dict(k=16, v=16, k_token=128, k_head=64, v_token=128, v_head=64, rotary=None, out_token=128, out_head=64, heads=4, ws=16,
                 nbytes=1 << 40, c=_address(c), b=_address(b))
        a.update(change)
        rotary = a["rotary"] and _gq_hip.Rotary(*a["rotary"])
        args = {"gq_kv_append_f16": (a["k"], a["k_token"], a["k_head"], a["v"], a["v_token"], a["v_head"], rotary and _address(rotary)),
                "gq_kv_gather_f16": (a["k"], a["v"]),
                "gq_kv_attention_f16": (a["k"], a["k_token"], a["k_head"], a["v"], a["out_token"], a["out_head"], a["heads"], 1.0, a["ws"], a["nbytes"])}
        return _refused(code, name, a["c"], a["b"], *args[name], None)

    for name in ("gq_kv_append_f16", "gq_kv_gather_f16", "gq_kv_attention_f16"):
        refused(GQ_ERR_NULL_POINTER, name, c=None)
        refused(GQ_ERR_NULL_POINTER, name, b=None)
        for i in range(4):
            refused(GQ_ERR_NULL_POINTER, name, cache=[(i, 0)])
            refused(GQ_ERR_MISALIGNED, name, cache=[(i, 8 if i < 2 else 18)])
        for i in range(3):
            refused(GQ_ERR_NULL_POINTER, name, batch=[(i, 0)])
            refused(GQ_ERR_MISALIGNED, name, batch=[(i, 18)])
        for i in (4, 5):
            refused(GQ_ERR_BAD_SHAPE, name, cache=[(i, -1)])
        for i in (3, 4, 5):
            refused(GQ_ERR_BAD_SHAPE, name, batch=[(i, -1)])
        for dim in (0, 8, 72, 272):
            assert "head_dim" in refused(GQ_ERR_UNSUPPORTED, name, cache=[(6, dim)])
        refused(GQ_ERR_UNSUPPORTED, name, cache=[(5, 1025)])
        refused(GQ_ERR_UNSUPPORTED, name, batch=[(5, (1 << 24) + 1)])
        refused(GQ_ERR_NULL_POINTER, name, k=0)
        refused(GQ_ERR_NULL_POINTER, name, v=0)
        refused(GQ_ERR_MISALIGNED, name, k=24)
    for name in ("gq_kv_append_f16", "gq_kv_attention_f16"):
        refused(GQ_ERR_MISALIGNED, name, k_token=129)
        refused(GQ_ERR_UNSUPPORTED, name, k_head=-64)
    refused(GQ_ERR_MISALIGNED, "gq_kv_append_f16", v=24)
    assert "gq_rotary_f16" in refused(GQ_ERR_UNSUPPORTED, "gq_kv_append_f16", rotary=(16, 1.0, 24, 1))
    refused(GQ_ERR_UNSUPPORTED, "gq_kv_append_f16", rotary=(16, 1.0, 12, 0))
    refused(GQ_ERR_BAD_SHAPE, "gq_kv_append_f16", rotary=(16, 1.0, 80, 0))
    for heads in (0, -4, 3):
        assert "q_heads" in refused(GQ_ERR_BAD_SHAPE, "gq_kv_attention_f16", heads=heads)
    refused(GQ_ERR_MISALIGNED, "gq_kv_attention_f16", v=17)
    refused(GQ_ERR_UNSUPPORTED, "gq_kv_attention_f16", out_head=-1)
    refused(GQ_ERR_NULL_POINTER, "gq_kv_attention_f16", ws=0)
    refused(GQ_ERR_MISALIGNED, "gq_kv_attention_f16", ws=24)
    need = _gq_hip.load().gq_kv_attention_workspace_bytes(64)
    assert need > 0 and "workspace" in refused(GQ_ERR_BAD_SHAPE, "gq_kv_attention_f16", nbytes=need - 1)
    assert _gq_hip.load().gq_kv_attention_workspace_bytes(72) == GQ_ERR_UNSUPPORTED


def test_adapter_refusals():
    lib = _gq_hip.load()
    good = [16, 16, 16, 4, 8, 64, 128]

    def adapters(*change):
        a = list(good)
        for i, value in change:
            a[i] = value
        return _gq_hip.Adapters(*a)

    ok = dict(plan=16, rows=5, x=16, xs=64, y=16, ys=128, out=32, os=128, act=0, ws=256, nbytes=1 << 40, dx=16, dxs=64, dxo=32, dxos=64, dd=16, du=16)

    def refused(code, name, *change, **values):
        a, v = adapters(*change), {**ok, **values}
        if name == "apply":
            args = (v["x"], v["xs"], v["y"], v["ys"], v["out"], v["os"], v["act"])
        else:
            args = (v["x"], v["xs"], v["y"], v["ys"], v["dx"], v["dxs"], v["dxo"], v["dxos"], v["dd"], v["du"])
        return _refused(code, f"gq_adapter_{name}_f16", _address(a), v["plan"], v["rows"], *args, v["ws"], v["nbytes"], None)

    for name in ("apply", "grad"):
        for i in range(3):
            refused(GQ_ERR_NULL_POINTER, name, (i, 0))
            refused(GQ_ERR_MISALIGNED, name, (i, 17))
        for i in range(3, 7):
            refused(GQ_ERR_BAD_SHAPE, name, (i, -1))
        for rank in (0, 129):
            assert "rank" in refused(GQ_ERR_UNSUPPORTED, name, (4, rank))
        for count in (0, 2049):
            assert "n_adapters" in refused(GQ_ERR_UNSUPPORTED, name, (3, count))
        refused(GQ_ERR_UNSUPPORTED, name, rows=(1 << 24) + 1)
        refused(GQ_ERR_BAD_SHAPE, name, rows=-1)
        refused(GQ_ERR_UNSUPPORTED, name, (5, 0))
        refused(GQ_ERR_NULL_POINTER, name, plan=0)
        refused(GQ_ERR_NULL_POINTER, name, x=0)
        refused(GQ_ERR_MISALIGNED, name, plan=24)
        refused(GQ_ERR_MISALIGNED, name, x=17)
        refused(GQ_ERR_UNSUPPORTED, name, xs=-1)
        refused(GQ_ERR_UNSUPPORTED, name, ys=(1 << 30) + 1)
        refused(GQ_ERR_NULL_POINTER, name, ws=0)
        refused(GQ_ERR_MISALIGNED, name, ws=128)
        need = getattr(lib, f"gq_adapter_{name}_workspace_bytes")(_address(adapters()), 5)
        assert need > 0 and "workspace" in refused(GQ_ERR_BAD_SHAPE, name, nbytes=need - 1)
    refused(GQ_ERR_UNSUPPORTED, "apply", act=9)
    refused(GQ_ERR_NULL_POINTER, "apply", out=0)
    assert "in place" in refused(GQ_ERR_UNSUPPORTED, "apply", out=16, os=136)
    refused(GQ_ERR_NULL_POINTER, "grad", y=0)
    refused(GQ_ERR_NULL_POINTER, "grad", dd=0)
    refused(GQ_ERR_MISALIGNED, "grad", du=18)
    refused(GQ_ERR_UNSUPPORTED, "grad", rows=0)
    assert "in place" in refused(GQ_ERR_UNSUPPORTED, "grad", dxo=16, dxos=72)
    _gq_hip.call("gq_adapter_apply_f16", _address(adapters((0, 0))), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, None)  # no rows
    need = lib.gq_adapter_plan_bytes(100, 4)
    assert need > 400
    assert lib.gq_adapter_plan_bytes(-1, 4) == GQ_ERR_BAD_SHAPE and lib.gq_adapter_plan_bytes(5, 2049) == GQ_ERR_UNSUPPORTED
    _refused(GQ_ERR_NULL_POINTER, "gq_adapter_plan", 0, 100, 4, 16, need, None)
    _refused(GQ_ERR_NULL_POINTER, "gq_adapter_plan", 16, 100, 4, 0, need, None)
    _refused(GQ_ERR_MISALIGNED, "gq_adapter_plan", 16, 100, 4, 24, need, None)
    _refused(GQ_ERR_BAD_SHAPE, "gq_adapter_plan", 16, 100, 4, 16, need - 1, None)
    _gq_hip.call("gq_adapter_plan", 0, 0, 4, 0, 0, None)


@pytest.mark.parametrize("x,dy", [(64, 16), (16, 64)])
def test_adapter_gradient_apart_from_what_it_reads(x, dy):
    """dx_out is written before the gradients of the weights read x and dy."""
    a = _gq_hip.Adapters(16, 16, 16, 4, 8, 64, 64)
    message = _refused(GQ_ERR_UNSUPPORTED, "gq_adapter_grad_f16", _address(a), 16, 5, x, 64, dy, 64, 32, 64, 64, 64, 16, 16, 256, 1 << 40, None)
    assert "dx_out must not be x or dy" in message


def test_frequencies():
    w, factor = rotary_frequencies(64)
    assert factor == 1 and w[0] == 1 and w.shape == (32,) and math.isclose(w[-1], 10000 ** (-62 / 64))
    assert np.allclose(rotary_frequencies(64, scaling=dict(kind="linear", factor=4))[0], w / 4, rtol=1e-15)
    ntk, _ = rotary_frequencies(64, scaling=dict(kind="ntk", factor=4))
    assert ntk[0] == 1 and math.isclose(ntk[-1], w[-1] / 4, rel_tol=1e-12)  # the slowest pair is stretched by the factor
    yarn, factor = rotary_frequencies(64, scaling=dict(kind="yarn", factor=8, original_length=4096))
    turns = 4096 * w / (2 * math.pi)
    assert math.isclose(factor, 0.1 * math.log(8) + 1)
    assert np.array_equal(yarn[turns >= 32], w[turns >= 32]) and np.allclose(yarn[turns <= 1], w[turns <= 1] / 8, rtol=1e-15)
    ramp = (turns > 1) & (turns < 32)
    assert ramp.any() and ((yarn < w) & (yarn > w / 8))[ramp].all()
    for bad in (dict(kind="other", factor=2), dict(kind="linear"), dict(kind="linear", factor=0.5), dict(kind="linear", factor=2, beta_fast=3),
                dict(kind="yarn", factor=2), dict(kind="yarn", factor=2, original_length=10, beta_fast=1, beta_slow=1)):
        with pytest.raises(ValueError):
            rotary_frequencies(64, scaling=bad)
    for rotary_dim in (0, 3, -2):
        with pytest.raises(ValueError):
            rotary_frequencies(rotary_dim)
    with pytest.raises(ValueError):
        rotary_frequencies(2, scaling=dict(kind="ntk", factor=2))
    with pytest.raises(ValueError):
        RotaryPosEmbed(64, layout="other", device="cpu")
    with pytest.raises(ValueError):
        RotaryPosEmbed(300, device="cpu")


def test_python_calls_refuse_cpu_tensors_types_and_shapes():
    rotary, half = RotaryPosEmbed(32, device="cpu"), torch.zeros((3, 2, 64), dtype=torch.float16)
    positions = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        rotary_pos_embed(half, positions, rotary)
    with pytest.raises(ValueError):
        rotary_pos_embed(half[0], positions, rotary)
    cache = KVCacheGQ(2, 2, 64, "cpu")
    batch = (torch.tensor([0, 3], dtype=torch.int32), torch.tensor([3], dtype=torch.int32), torch.zeros((1, 1), dtype=torch.int32))
    with pytest.raises(RuntimeError):
        kv_cache_append(cache, half, half, *batch)
    with pytest.raises(RuntimeError):
        kv_cache_attention(half, cache, *batch)
    for dim in (0, 8, 65, 272):
        with pytest.raises(ValueError):
            KVCacheGQ(2, 2, dim, "cpu")
    with pytest.raises(ValueError):
        KVCacheGQ.from_tensors(cache.k_codes[..., :32].contiguous(), cache.v_codes, cache.k_scale, cache.v_scale)
    with pytest.raises(TypeError):
        KVCacheGQ.from_tensors(cache.k_codes.char(), cache.v_codes, cache.k_scale, cache.v_scale)
    with pytest.raises(TypeError):
        KVCacheGQ.from_tensors(cache.k_codes, cache.v_codes, cache.k_scale.double(), cache.v_scale)
    with pytest.raises(ValueError):
        KVCacheGQ.from_tensors(cache.k_codes, cache.v_codes, cache.k_scale[:1], cache.v_scale)
    down, up = torch.zeros((2, 8, 64), dtype=torch.float16), torch.zeros((2, 96, 8), dtype=torch.float16)
    adapters = LowRankAdapters(down, up, 2.0)
    assert (adapters.rank, adapters.in_features, adapters.out_features) == (8, 64, 96) and adapters.scaling.tolist() == [2, 2]
    for bad in ((down, up[:1]), (down, up.transpose(1, 2)), (down[0], up[0]), (torch.zeros((2, 129, 4), dtype=torch.float16), torch.zeros((2, 4, 129), dtype=torch.float16))):
        with pytest.raises(ValueError):
            LowRankAdapters(*bad)
    with pytest.raises(TypeError):
        LowRankAdapters(down.float(), up)
    with pytest.raises(ValueError):
        LowRankAdapters(down, up, torch.zeros(3))
    with pytest.raises(RuntimeError):
        AdapterPlan(torch.zeros(3, dtype=torch.int32), 2)
    layer, x = LinearGQ(96, group_size=32), torch.zeros((3, 64), dtype=torch.float16)
    with pytest.raises(ValueError):
        layer.build(x, adapters=adapters)
    with pytest.raises(ValueError):
        layer.build(x[:, :32], adapters=adapters, plan=object())
    with pytest.raises(ValueError):
        layer.grad(x)
    with pytest.raises(ValueError):
        low_rank_adapters(x, x, adapters, plan=type("Plan", (), dict(n_adapters=3, device=adapters.device, rows=3))())


@pytest.mark.parametrize("rows,k,n", [(3, 64, 0), (0, 64, 32), (3, 0, 32)])
@pytest.mark.parametrize("with_dx", [False, True])
def test_gradients_without_rows_or_features(monkeypatch, rows, k, n, with_dx):
    """No dx stands for zeros, also where there is nothing to add to them.  (These sizes launch nothing: CPU tensors do, once the
    check for GPU ones is taken away; new memory is filled with NaN.)"""
    module = sys.modules["popxl_addons.ops.low_rank_adapters.low_rank_adapters"]
    monkeypatch.setattr(module, "_matrix", lambda name, t, *rest: t)
    adapters = LowRankAdapters(torch.ones((2, 4, k), dtype=torch.float16), torch.ones((2, n, 4), dtype=torch.float16))
    plan = type("Plan", (), dict(n_adapters=2, device=adapters.device, index=adapters.index, rows=rows))()
    x, dy = torch.ones((rows, k), dtype=torch.float16), torch.ones((rows, n), dtype=torch.float16)
    dx = torch.full((rows, k), 2.0, dtype=torch.float16) if with_dx else None
    torch.use_deterministic_algorithms(True)
    try:
        got, d_down, d_up = module.low_rank_adapters_grad(x, dy, adapters, plan, dx=dx)
    finally:
        torch.use_deterministic_algorithms(False)
    assert torch.equal(got, torch.zeros_like(x) if dx is None else dx) and got is not dx
    assert d_down.dtype == d_up.dtype == torch.float32 and not d_down.any() and not d_up.any()


def test_attention_apart_from_its_queries():
    """Several workgroups read a row of q when others have written the result there."""
    cache, batch = _gq_hip.KvCache(16, 16, 16, 16, 10, 2, 64), _gq_hip.KvBatch(16, 16, 16, 3, 4, 5)
    for token_stride, head_stride in ((256, 64), (64, 320)):  # (the same start is the same first row, whatever the strides)
        message = _refused(GQ_ERR_UNSUPPORTED, "gq_kv_attention_f16", _address(cache), _address(batch), 16, 256, 64, 16, token_stride, head_stride,
                           4, 1.0, 16, 1 << 40, None)
        assert "out must not be q" in message


def test_results_whose_rows_lie_on_each_other():
    """A result that is one row many times (an expanded tensor) would hold whatever came last."""
    rotary = _address(_gq_hip.Rotary(16, 1.0, 32, 0))
    for t, o in (((64, 32), (0, 32)), ((64, 32), (32, 0)), ((0, 32), (0, 32))):
        out = 16 if t == o else 32
        assert "on each other" in _refused(GQ_ERR_UNSUPPORTED, "gq_rotary_f16", 16, *t, 16, rotary, 0, out, *o, 3, 2, 32, None)
    cache, batch = _address(_gq_hip.KvCache(16, 16, 16, 16, 10, 2, 64)), _address(_gq_hip.KvBatch(16, 16, 16, 3, 4, 5))
    for o in ((0, 64), (256, 0)):
        assert "on each other" in _refused(GQ_ERR_UNSUPPORTED, "gq_kv_attention_f16", cache, batch, 16, 256, 64, 32, *o, 4, 1.0, 16, 1 << 40, None)
    adapters = _address(_gq_hip.Adapters(16, 16, 16, 4, 8, 64, 128))
    for stride in (0, 120):
        assert "on each other" in _refused(GQ_ERR_UNSUPPORTED, "gq_adapter_apply_f16", adapters, 16, 5, 16, 64, 16, 128, 32, stride, 0, 256, 1 << 40, None)
    for stride in (0, 63):
        assert "on each other" in _refused(GQ_ERR_UNSUPPORTED, "gq_adapter_grad_f16", adapters, 16, 5, 16, 64, 16, 128, 64, 64, 32, stride, 16, 16, 256,
                                           1 << 40, None)
    k = _address(_gq_hip.KvCache(16, 16, 16, 16, 10, 2, 64))
    assert "on each other" in _refused(GQ_ERR_UNSUPPORTED, "gq_kv_gather_f16", k, batch, 16, 16, None)


def test_strides_of_single_rows_do_not_matter():
    fake = 1 << 20
    cache = ["KvCache", fake, fake, fake, fake, 10, 2, 64]
    calls = [[0, "gq_rotary_f16", [fake, 0, 32, fake, ["Rotary", fake, 1.0, 32, 0], 0, 2 * fake, 0, 32, 1, 2, 32, None]],
             [0, "gq_rotary_f16", [fake, 32, 0, fake, ["Rotary", fake, 1.0, 32, 0], 0, 2 * fake, 32, 0, 5, 1, 32, None]],
             [0, "gq_kv_attention_f16", [cache, ["KvBatch", fake, fake, fake, 1, 4, 1], fake, 0, 64, 2 * fake, 0, 64, 2, 1.0, fake, 1 << 40, None]],
             [0, "gq_adapter_apply_f16", [["Adapters", fake, fake, fake, 4, 8, 64, 128], fake, 1, fake, 64, fake, 128, 2 * fake, 0, 0, fake, 1 << 40, None]]]
    for call, result in zip(calls, launches(calls)):
        assert result["code"] == 0 and result["records"], call


def test_rotary_of_given_frequencies():
    """Frequencies of the caller's own (another way to stretch a context, say) instead of base and scaling."""
    w, factor = rotary_frequencies(64, base=500.0, scaling=dict(kind="yarn", factor=8, original_length=4096))
    made = RotaryPosEmbed(64, base=500.0, layout="half", scaling=dict(kind="yarn", factor=8, original_length=4096), device="cpu")
    for frequencies in (w, w.tolist(), torch.from_numpy(w)):
        given = RotaryPosEmbed.from_frequencies(frequencies, factor, layout="half", device="cpu")
        assert torch.equal(given.turns, made.turns) and (given.rotary_dim, given.factor, given.layout) == (64, made.factor, "half")
        assert bytes(given._c)[8:] == bytes(made._c)[8:]
    single = RotaryPosEmbed.from_frequencies(np.float32([0.5, -0.25, 0]), device="cpu")  # backwards, and not at all
    assert single.turns.dtype == torch.float64 and np.array_equal(single.turns.numpy() * 2 * math.pi, [0.5, -0.25, 0]) and single.factor == 1
    for bad in ([], [[1.0, 2.0]], 1.0, [1.0] * 129, [1.0, math.nan], [math.inf], [1j]):
        with pytest.raises(ValueError):
            RotaryPosEmbed.from_frequencies(bad, device="cpu")
    for factor in (math.nan, math.inf):
        with pytest.raises(ValueError):
            RotaryPosEmbed.from_frequencies([1.0], factor, device="cpu")
    with pytest.raises(ValueError):
        RotaryPosEmbed.from_frequencies([1.0], layout="other", device="cpu")


def test_yarn_ramp_is_linear_in_turns():
    """Between the pairs that are kept and those that are stretched: (turns - beta_slow) / (beta_fast - beta_slow) is what stays of w."""
    w, _ = rotary_frequencies(128, base=1e6)
    for fast, slow in ((32, 1), (20, 4)):
        yarn, _ = rotary_frequencies(128, base=1e6, scaling=dict(kind="yarn", factor=4, original_length=2048, beta_fast=fast, beta_slow=slow))
        for i in range(64):
            turns = 2048 * w[i] / (2 * math.pi)
            stays = min(max((turns - slow) / (fast - slow), 0), 1)
            assert math.isclose(yarn[i], w[i] * stays + w[i] / 4 * (1 - stays), rel_tol=1e-14)


class _Placed(torch.Tensor):
    """A host tensor that says it lies on the GPU `index`."""

    index = 0
    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", self.index))

    def get_device(self):
        return self.index


class _PlacedElsewhere(_Placed):
    index = 1


@pytest.mark.parametrize("dim", [0, -1])
def test_layer_on_another_device_than_its_input(dim):
    """The kernels would read the weight's address on the input's device."""
    layer = LinearGQ(64, group_size=32, dim=dim)
    layer.init_variables(64, torch.float16, "cpu")
    x = torch.zeros((3, 64), dtype=torch.float16).as_subclass(_Placed)
    for where in ("cpu", "cuda:1"):
        if where != "cpu":
            for name in ("weight_compressed", "weight_decompression_scale", "weight_decompression_bias", "bias"):
                layer.variables[name].data = layer.variables[name].data.as_subclass(_PlacedElsewhere)
        for call in (layer.build, layer.grad):
            with pytest.raises(ValueError, match=f"the layer is on {where}"):
                call(x)
