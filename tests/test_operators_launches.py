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
