"""What the operators beside the projections launch: limits of LDS that no call changes for another one."""
from collections import defaultdict

from launch_recorder import launches

FAKE = 1 << 20  # an address that nothing reads


def append(tokens, sequences, heads, dim, rotary_dim=0, device=0):
    cache = ["KvCache", FAKE, FAKE, FAKE, FAKE, 10, heads, dim]
    batch = ["KvBatch", FAKE, FAKE, FAKE, sequences, 4, tokens]
    rotary = ["Rotary", FAKE, 1.0, rotary_dim, 0] if rotary_dim else None
    return [device, "gq_kv_append_f16", [cache, batch, FAKE, heads * dim, dim, FAKE, heads * dim, dim, rotary, None]]


def attend(tokens, sequences, heads, dim, q_heads, width=4, device=0):
    cache = ["KvCache", FAKE, FAKE, FAKE, FAKE, 10, heads, dim]
    batch = ["KvBatch", FAKE, FAKE, FAKE, sequences, width, tokens]
    return [device, "gq_kv_attention_f16", [cache, batch, FAKE, q_heads * dim, dim, 2 * FAKE, q_heads * dim, dim, q_heads, 1.0, FAKE, 1 << 40, None]]


def plan(rows, adapters, device=0):
    return [device, "gq_adapter_plan", [FAKE, rows, adapters, FAKE, 1 << 40, None]]


def test_limits_of_lds_are_the_same_for_every_call():
    """The limit belongs to a kernel and a device, not to a call: a call that lowered it would have another thread's launch refused.
    So each is set to one value, once, before the first launch that needs it."""
    sizes = [append(1, 1, 2, 256, 256), append(64, 1, 2, 256, 256), append(200, 3, 2, 256, 256), append(200, 3, 2, 128, 128),
             append(40, 1, 2, 256, 256), append(70, 40, 2, 256, 256), append(70, 40, 2, 192, 192), append(500, 1, 1, 256),
             plan(100, 2048), plan(100, 1100), plan(100, 1023), plan(100, 1500), plan(100, 3),
             attend(1, 1, 1, 256, 1), attend(300, 1, 1, 256, 1), attend(1, 1, 1, 128, 1), attend(300, 1, 2, 128, 4), attend(300, 1, 2, 64, 4)]
    calls = [[device, *call[1:]] for device in (0, 3, 0) for call in sizes + sizes[::-1]]
    limits, most = defaultdict(list), defaultdict(int)
    for call, result in zip(calls, launches(calls)):
        assert result["code"] == 0, call
        assert any(r["launch"] for r in result["records"])
        for r in result["records"]:
            key = r["kernel"], r["device"]
            assert r["device"] == call[0] and r["kernel"] != "?"
            if not r["launch"]:
                limits[key].append(r["lds"])
            elif r["lds"] > 60 << 10:  # (what a kernel may use without asking is 64 KiB with its static arrays)
                assert limits[key] and limits[key][0] >= r["lds"], (call, r)
                most[key] = max(most[key], r["lds"])
    assert {device for _, device in limits} == {0, 3} and len(limits) >= 2 * 5
    for key, values in limits.items():
        assert len(values) == 1, (key, values)
        assert most[key] <= values[0] <= 160 << 10


def rotary(tokens, heads, dim, rotary_dim, device=0):
    return [device, "gq_rotary_f16", [FAKE, heads * dim, dim, FAKE, ["Rotary", FAKE, 1.0, rotary_dim, 0], 0, 2 * FAKE, heads * dim, dim, tokens, heads, dim, None]]


def gather(tokens, sequences, heads, dim, device=0):
    cache = ["KvCache", FAKE, FAKE, FAKE, FAKE, 10, heads, dim]
    return [device, "gq_kv_gather_f16", [cache, ["KvBatch", FAKE, FAKE, FAKE, sequences, 4, tokens], FAKE, 2 * FAKE, None]]


def adapters(rows, count, rank, k, n, grad, device=0):
    w = ["Adapters", FAKE, FAKE, FAKE, count, rank, k, n]
    if grad:
        return [device, "gq_adapter_grad_f16", [w, FAKE, rows, FAKE, k, 3 * FAKE, n, None, 0, 2 * FAKE, k, FAKE, FAKE, FAKE, 1 << 62, None]]
    return [device, "gq_adapter_apply_f16", [w, FAKE, rows, FAKE, k, 3 * FAKE, n, 2 * FAKE, n, 0, FAKE, 1 << 62, None]]


MOST = 1 << 24  # tokens, rows
UNSUPPORTED = -4
LARGEST = [
    rotary(MOST, 1, 16, 16), rotary(MOST - 1, 65535, 64, 32), rotary(MOST, 40, 128, 128), rotary((1 << 23) + 1, 3, 33, 2), rotary(1, 65535, 2048, 256),
    append(MOST, 1, 1, 128, 128), append(MOST, 1, 8, 128), append(MOST, 1 << 20, 1, 16), append(1 << 20, 1 << 20, 1, 64), gather(MOST, 1, 8, 128),
    attend(MOST, 1, 1, 128, 1), attend(1 << 20, 1 << 20, 1, 64, 8), attend(1 << 14, 1, 1024, 16, 65536 - 1024, 1 << 24), attend(1 << 14, 1 << 14, 8, 256, 32, 1 << 20),
    plan(MOST, 2048), plan(MOST, 1),
    *(adapters(rows, count, rank, k, n, grad) for grad in (False, True)
      for rows, count, rank, k, n in ((MOST, 2048, 128, 4096, 4096), (MOST, 1, 8, 4097, 33), (8191, 2048, 16, 1 << 20, 1 << 20), (1, 2048, 1, 1 << 20, 1))),
]


def test_largest_sizes_fit_a_grid():
    """Whatever is not refused is launched as grids that exist: fewer than 2^32 threads an axis, 65535 workgroups along y and z."""
    for call, result in zip(LARGEST, launches(LARGEST)):
        assert result["code"] in (0, UNSUPPORTED), (call, result["code"])
        assert bool(result["records"]) == (result["code"] == 0), call
        for r in result["records"]:
            if r["launch"]:
                assert all(0 < g and g * b < 1 << 32 for g, b in zip(r["grid"], r["block"])), (call, r)
                assert r["grid"][1] <= 65535 and r["grid"][2] <= 65535, (call, r)


def test_rotary_takes_as_many_tokens_as_it_says():
    calls = [rotary(tokens, 3, 64, 32) for tokens in (1, 511, MOST // 2, MOST // 2 + 1, MOST - 1, MOST)]
    for call, result in zip(calls, launches(calls)):
        assert result["code"] == 0
        assert sum(r["grid"][0] for r in result["records"]) == call[2][9]
    assert launches([rotary(MOST + 1, 1, 64, 32)])[0]["code"] == UNSUPPORTED
