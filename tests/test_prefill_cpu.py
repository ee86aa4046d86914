"""The plan of a packed batch and the refusals of the prefill operators, on the host."""
import ctypes

import pytest
import torch

from palu_b200 import _lib, build, prefill

ROW = ("q0", "npos", "vis0", "k0", "kvh", "t0", "t1", "slot")


def plan(q_lens, k_lens, n_q, n_kv, ctas=148, rows=None):
    build.build()
    lib, n = _lib.load(), len(q_lens)
    arr = lambda x: None if x is None else (ctypes.c_int32 * n)(*x)
    info = _lib.PrefillPlanInfo()
    _lib.check(lib.palu_plan_prefill(arr(q_lens), arr(k_lens), arr(rows), n, n_q, n_kv, ctas, None, 0, ctypes.byref(info)))
    buf = torch.zeros(max(1, info.bytes), dtype=torch.uint8)
    st = lib.palu_plan_prefill(arr(q_lens), arr(k_lens), arr(rows), n, n_q, n_kv, ctas, buf.data_ptr(), info.bytes - 1, ctypes.byref(info))
    assert st == _lib.PALU_ERR_WORKSPACE and "smaller" in lib.palu_last_error().decode()
    _lib.check(lib.palu_plan_prefill(arr(q_lens), arr(k_lens), arr(rows), n, n_q, n_kv, ctas, buf.data_ptr(), info.bytes, ctypes.byref(info)))
    part = lambda off, count: buf[off:off + 4 * count].view(torch.int32)
    start = part(info.off_start, info.n_ctas + 1).tolist()
    pieces = [dict(zip(ROW, p)) for p in part(info.off_pieces, 8 * info.n_pieces).view(-1, 8).tolist()]
    merges = part(info.off_merges, 6 * info.n_merges).view(-1, 6).tolist()
    tiles = part(info.off_tiles, 4 * info.n_tiles).view(-1, 4).tolist()
    return info, start, pieces, merges, tiles


@pytest.mark.parametrize("q_lens,k_lens,n_q,n_kv", [
    ([1], [1], 4, 1), ([5, 0, 300], [5, 9, 300], 32, 8), ([50], [20], 4, 4), ([64, 1], [9000, 20000], 8, 2),
    ([7], [0], 6, 2), ([], [], 8, 2), ([1000, 3], [1000, 3], 128, 1),
])
def test_every_query_tile_is_covered_once(q_lens, k_lens, n_q, n_kv):
    info, start, pieces, merges, tiles = plan(q_lens, k_lens, n_q, n_kv)
    ppt = 128 // (n_q // n_kv)
    assert info.n_ctas <= 148 and start[0] == 0 and start[-1] == len(pieces) and sorted(start) == start
    want, q0, k0 = {}, 0, 0
    for ql, kl in zip(q_lens, k_lens):
        for a in range(0, ql, 2 * ppt):
            n, vis0 = min(2 * ppt, ql - a), kl - ql + a + 1
            for h in range(n_kv):
                want[q0 + a, h] = (n, vis0, k0, -(-max(0, vis0 + n - 1) // 128))
        q0, k0 = q0 + ql, k0 + kl
    got = {}
    for p in pieces:
        assert (p["npos"], p["vis0"], p["k0"]) == want[p["q0"], p["kvh"]][:3]
        got.setdefault((p["q0"], p["kvh"]), []).append((p["t0"], p["t1"], p["slot"]))
    joined = {(m[0], m[3]): m for m in merges}
    assert set(got) == set(want) and sorted(p["slot"] for p in pieces if p["slot"] >= 0) == list(range(info.n_slots))
    for key, parts in got.items():
        parts.sort()
        assert parts[0][0] == 0 and parts[-1][1] == want[key][3]
        assert all(x[1] == y[0] for x, y in zip(parts, parts[1:]))
        if len(parts) == 1:
            assert parts[0][2] == -1 and key not in joined
        else:
            m = joined[key]
            assert sorted(x[2] for x in parts) == list(range(m[4], m[4] + m[5]))
    # 128-token tiles of the cached rows, for the rebuild
    at = 0
    for t in sorted(tiles, key=lambda t: t[2]):
        assert t[2] == at and 0 < t[3] <= 128
        at += t[3]
    assert at == sum(k_lens)


def test_long_keys_behind_few_queries_are_split():
    info, *_ = plan([64], [32768], 8, 2)
    assert info.n_merges == 2 and info.n_slots > 100      # both KV heads, over most of the SMs
    assert plan([4096], [4096], 32, 8)[0].n_merges == 0   # enough query tiles: whole items


def test_cache_rows_reach_the_rebuild_tiles():
    tiles = plan([0, 0], [140, 3], 4, 4, rows=[5, 2])[4]
    assert tiles == [[5, 0, 0, 128], [2, 0, 140, 3], [5, 128, 128, 12]]


@pytest.mark.parametrize("args,needle", [
    (([1], [1], 30, 8), "must divide"), (([1], [1], 129, 1), "128 query heads"), (([-1], [1], 4, 1), "negative"),
    (([1], [-2], 4, 1), "negative"), (([1 << 28, 1], [1, 1], 4, 1), "packed tokens"),
])
def test_plan_refusals(args, needle):
    with pytest.raises(RuntimeError, match=needle):
        plan(*args)


def test_plan_class_refusals():
    with pytest.raises(RuntimeError, match="same length"):
        prefill.PrefillPlan([1, 2], [1], n_q_heads=4, n_kv_heads=1)
    with pytest.raises(RuntimeError, match="one cache row per sequence"):
        prefill.PrefillPlan([1, 2], rows=[0], n_q_heads=4, n_kv_heads=1)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        prefill.PrefillPlan([1], n_q_heads=4, n_kv_heads=1, device="cpu")
    with pytest.raises(RuntimeError, match="32 bits"):
        prefill.PrefillPlan([1 << 40], n_q_heads=4, n_kv_heads=1)


def _call(info, **kw):
    a = dict(q=16, qs=(512, 128), k=16, ks=(128, 128), v=16, vs=(64, 64), out=16, d_v=64, data=16, ws=None, wsb=0, scale=1.0)
    a.update(kw)
    lib = _lib.load()
    st = lib.palu_prefill_attn(a["q"], *a["qs"], a["k"], *a["ks"], a["v"], *a["vs"], a["out"], a["d_v"], ctypes.byref(info),
                               a["data"], a["ws"], a["wsb"], a["scale"], None)
    return st, lib.palu_last_error().decode()


@pytest.mark.parametrize("change,needle", [
    (dict(d_v=0), "d_v"), (dict(d_v=24), "d_v"), (dict(d_v=144), "d_v"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(q=None), "must be set"),
    (dict(v=None), "must be set"), (dict(q=8), "aligned"), (dict(out=20), "aligned"), (dict(ks=(130, 128)), "strides"),
    (dict(vs=(64, 0)), "strides"), (dict(data=None), "plan"),
])
def test_attention_refusals_come_before_any_launch(change, needle):
    """The pointers are dummies: validation fails first."""
    info = plan([4], [4], 4, 1)[0]
    st, msg = _call(info, **change)
    assert st == _lib.PALU_ERR_INVALID and needle in msg, msg


def test_attention_refuses_a_missing_workspace():
    info = plan([64], [32768], 8, 2)[0]
    need = _lib.load().palu_prefill_workspace_bytes(ctypes.byref(info), 64)
    assert need == info.n_slots * 256 * 66 * 4
    st, msg = _call(info, qs=(1024, 128), ks=(256, 128), vs=(128, 64), ws=16, wsb=need - 1)
    assert st == _lib.PALU_ERR_WORKSPACE and "workspace" in msg


def test_cpu_tensors_are_refused():
    q = torch.zeros(4, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        prefill.prefill_attn(q, q, q, None)


def test_limits_of_the_largest_calls():
    with pytest.raises(RuntimeError, match="work items"):
        plan([1 << 28], [1], 1024, 8)                     # 2^27 query tiles x 8 KV heads
    with pytest.raises(RuntimeError, match="65536 query heads"):
        plan([1], [1], 1 << 17, 1 << 17)
    st, msg = _call(plan([4], [4], 4, 1)[0], scale=3e38)  # finite, but not times log2 e
    assert st == _lib.PALU_ERR_INVALID and "scale" in msg
