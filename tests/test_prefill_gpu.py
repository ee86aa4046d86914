"""Packed causal prefill attention on the GPU (palu_plan_prefill, palu_prefill_attn) against the formula in 64 bits.

Tolerance, per element, from the roundings of the kernel (w_j the softmax weights, A = sum_j w_j |v_j|):
* each probability is rounded to bf16 before the second product: at most 2^-8 of it, together 2^-8 A;
* the result is rounded to bf16 once: 2^-8 |o|;
* scores accumulate in fp32 (128 products, |q . k| of a few tens) and the exponential is good to 2^-12 or better,
  sums in fp32: together below 2^-11 A.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

H = 128


def formula(q, k, v, q_lens, k_lens, scale):
    """(o, A) in float64; masked keys and values are never touched."""
    n_q, n_kv, d = q.shape[1], k.shape[1], v.shape[2]
    rep = n_q // n_kv
    o = torch.zeros(q.shape[0], n_q, d, dtype=torch.float64)
    A = torch.zeros_like(o)
    q0 = k0 = 0
    for ql, kl in zip(q_lens, k_lens):
        for i in range(ql):
            n = min(kl, max(0, i + kl - ql + 1))
            if n:
                ks, vs = k[k0:k0 + n].double(), v[k0:k0 + n].double()
                x = torch.einsum("grd,ngd->grn", q[q0 + i].double().view(n_kv, rep, H), ks) * scale
                w = torch.softmax(x, -1)
                o[q0 + i] = torch.einsum("grn,ngd->grd", w, vs).reshape(n_q, d)
                A[q0 + i] = torch.einsum("grn,ngd->grd", w, vs.abs()).reshape(n_q, d)
        q0, k0 = q0 + ql, k0 + kl
    return o, A


def inputs(q_lens, k_lens, n_q, n_kv, d_v, seed=0, q_scale=1.0):
    g = torch.Generator().manual_seed(seed)
    bf = torch.bfloat16
    q = (torch.randn(sum(q_lens), n_q, H, generator=g) * q_scale).to(bf)
    return q, torch.randn(sum(k_lens), n_kv, H, generator=g).to(bf), torch.randn(sum(k_lens), n_kv, d_v, generator=g).to(bf)


def check(got, q, k, v, q_lens, k_lens, scale=H ** -0.5):
    o, A = formula(q, k, v, q_lens, k_lens, scale)
    bad = (got.double().cpu() - o).abs() > 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -11) * A
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} elements out of tolerance, first at {bad.nonzero()[0].tolist()}"


def attend(cuda, q, k, v, q_lens, k_lens, **kw):
    from palu_b200 import prefill
    plan = prefill.PrefillPlan(q_lens, k_lens, n_q_heads=q.shape[1], n_kv_heads=k.shape[1], device=cuda)
    out = prefill.prefill_attn(q.to(cuda), k.to(cuda), v.to(cuda), plan, **kw)
    torch.cuda.synchronize()
    assert plan.status() == 0, "a bounded device wait expired"
    return out


CASES = [
    # q_lens, k_lens, n_q, n_kv, d_v
    ([1], [1], 4, 1, 64),
    ([1], [300], 32, 8, 128),
    ([5, 0, 64], [5, 0, 64], 8, 2, 64),
    ([1, 17, 33, 128], [1, 17, 33, 128], 8, 2, 64),
    ([65, 129, 2], [65, 129, 2], 4, 4, 128),          # one head per KV head: 128 positions per chain
    ([127, 255, 256, 257], [127, 255, 256, 257], 8, 8, 128),
    ([200, 31], [457, 31], 6, 2, 96),                 # three heads per KV head: rows without a position
    ([70], [70], 10, 2, 48),
    ([40, 3], [40, 700], 8, 1, 16),
    ([9, 20], [9, 20], 128, 1, 80),                   # 128 heads per KV head: one position per chain
    ([50], [20], 4, 1, 64),                           # the first 30 queries see nothing
    ([300, 10], [100, 0], 4, 2, 128),                 # whole tiles of queries see nothing; a sequence without keys
    ([130], [2000], 4, 1, 112),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"q{'_'.join(map(str, c[0]))}-k{'_'.join(map(str, c[1]))}-h{c[2]}_{c[3]}-d{c[4]}")
def test_matches_the_formula(cuda, case):
    q_lens, k_lens, n_q, n_kv, d_v = case
    q, k, v = inputs(q_lens, k_lens, n_q, n_kv, d_v)
    check(attend(cuda, q, k, v, q_lens, k_lens), q, k, v, q_lens, k_lens)


@pytest.mark.parametrize("d_v", [64, 128])
def test_scores_that_outgrow_the_running_reference(cuda, d_v):
    """Key norms that rise along the sequence move the rows' maxima by far more than the rescale threshold."""
    q, k, v = inputs([150], [900], 4, 1, d_v, seed=3, q_scale=4.0)
    k = (k.float() * torch.linspace(0.02, 6.0, 900)[:, None, None]).to(torch.bfloat16)
    check(attend(cuda, q, k, v, [150], [900]), q, k, v, [150], [900])


def test_scale_is_applied(cuda):
    q, k, v = inputs([33], [70], 4, 2, 32, seed=4)
    check(attend(cuda, q, k, v, [33], [70], scale=0.5), q, k, v, [33], [70], scale=0.5)


@pytest.mark.parametrize("d_v", [64, 128])
def test_what_is_masked_does_not_reach_the_result(cuda, d_v):
    """NaN and infinities in later tokens of the same prompt, and in the next sequence of the batch."""
    q_lens = k_lens = [100, 37]
    q, k, v = inputs(q_lens, k_lens, 8, 2, d_v, seed=5)
    want, _ = formula(q, k, v, q_lens, k_lens, H ** -0.5)
    k2, v2 = k.clone(), v.clone()
    for t, x in ((60, math.nan), (61, math.inf), (80, -math.inf), (100, math.nan), (136, math.inf)):
        k2[t] = x
        v2[t] = x
    got = attend(cuda, q, k2, v2, q_lens, k_lens).double().cpu()
    clean = attend(cuda, q, k, v, q_lens, k_lens).double().cpu()
    assert torch.equal(got[:60], clean[:60])               # queries before the first bad token: bit for bit
    assert torch.isnan(got[60:100]).all() and torch.isnan(got[100:]).all()


def test_non_finite_values_reach_exactly_the_rows_that_see_them(cuda):
    q_lens = k_lens = [90, 5]
    q, k, v = inputs(q_lens, k_lens, 4, 2, 64, seed=6)
    v2 = v.clone()
    v2[70, 0, 3], v2[75, 0, 3], v2[72, 1, 63] = math.inf, -math.inf, math.nan
    got = attend(cuda, q, k, v2, q_lens, k_lens).float().cpu()
    clean = attend(cuda, q, k, v, q_lens, k_lens).float().cpu()
    want = clean.clone()
    want[70:75, 0:2, 3] = math.inf                         # heads 0, 1 read KV head 0
    want[75:90, 0:2, 3] = math.nan
    want[72:90, 2:4, 63] = math.nan
    assert torch.equal(torch.nan_to_num(got, nan=7e30, posinf=8e30), torch.nan_to_num(want, nan=7e30, posinf=8e30))


def test_a_score_row_of_minus_infinities_is_nan_and_an_unseeing_row_is_zero(cuda):
    q, k, v = inputs([3], [2], 4, 1, 64, seed=7)
    k[:] = 0
    k[..., 0] = -math.inf
    q[..., 0] = 1.0
    got = attend(cuda, q, k, v, [3], [2]).float().cpu()
    assert (got[0] == 0).all() and torch.isnan(got[1:]).all()


def test_rows_behind_the_batch_and_strided_inputs(cuda):
    """q, k and v as slices of one projection; `out` is the front of a larger buffer whose rest stays as it was."""
    from palu_b200 import prefill
    lens = [45, 20]
    q, k, v = inputs(lens, lens, 8, 2, 48, seed=8)
    wide = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1).to(cuda)
    qs = wide[:, :1024].unflatten(1, (8, 128))
    ks = wide[:, 1024:1280].unflatten(1, (2, 128))
    vs = wide[:, 1280:].unflatten(1, (2, 48))
    assert not qs.is_contiguous()
    plan = prefill.PrefillPlan(lens, n_q_heads=8, n_kv_heads=2, device=cuda)
    buf = torch.full((80, 8, 48), 5.0, dtype=torch.bfloat16, device=cuda)
    out = prefill.prefill_attn(qs, ks, vs, plan, out=buf[:65])
    check(out, q, k, v, lens, lens)
    assert (buf[65:] == 5).all()


def test_one_plan_on_two_streams_and_in_two_graphs(cuda):
    """A plan whose work is split along the keys (partial results), used by overlapping calls and captured twice."""
    from palu_b200 import prefill
    q_lens, k_lens = [20], [6000]
    a = [x.to(cuda) for x in inputs(q_lens, k_lens, 8, 2, 64, seed=9)]
    b = [x.to(cuda) for x in inputs(q_lens, k_lens, 8, 2, 64, seed=10)]
    plan = prefill.PrefillPlan(q_lens, k_lens, n_q_heads=8, n_kv_heads=2, device=cuda)
    assert plan.workspace_bytes(64) > 0
    want = [prefill.prefill_attn(*x, plan) for x in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, x in zip(streams, (a, b)):
        with torch.cuda.stream(s):
            got.append([prefill.prefill_attn(*x, plan) for _ in range(5)])
    graphs, outs = [], []
    torch.cuda.synchronize()
    for x in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(prefill.prefill_attn(*x, plan))
        graphs.append(g)
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for w, xs, o in zip(want, got, outs):
        assert all(torch.equal(w, x) for x in xs) and torch.equal(w, o)
    assert plan.status() == 0


def test_results_do_not_depend_on_the_other_sequences(cuda):
    """A prompt alone and inside a batch: the same bits (no atomics, the order of its tiles is its own)."""
    q, k, v = inputs([77], [77], 8, 2, 64, seed=11)
    alone = attend(cuda, q, k, v, [77], [77])
    q2, k2, v2 = inputs([5, 77, 40], [5, 77, 40], 8, 2, 64, seed=12)
    q2[5:82], k2[5:82], v2[5:82] = q, k, v
    assert torch.equal(attend(cuda, q2, k2, v2, [5, 77, 40], [5, 77, 40])[5:82], alone)


def test_long_prompt_against_the_formula_at_its_ends(cuda):
    """4500 tokens (many tiles, several pieces): sampled query rows against the formula."""
    n = 4500
    q, k, v = inputs([n], [n], 4, 2, 128, seed=13)
    got = attend(cuda, q, k, v, [n], [n]).cpu()
    for i in (0, 1, 127, 128, 2047, 4096, 4498, 4499):
        o, A = formula(q[i:i + 1], k[:i + 1], v[:i + 1], [1], [i + 1], H ** -0.5)
        err = (got[i:i + 1].double() - o).abs()
        assert (err <= 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -11) * A).all(), i


def test_an_expired_wait_gives_nan_and_a_status(cuda):
    from palu_b200 import _lib, prefill
    q, k, v = (x.to(cuda) for x in inputs([30], [30], 8, 2, 64, seed=14))
    plan = prefill.PrefillPlan([30], n_q_heads=8, n_kv_heads=2, device=cuda)
    want = prefill.prefill_attn(q, k, v, plan)
    _lib.set_wait_limit(2_000_000, True)                    # 2 ms; the producer loads no V
    try:
        out = prefill.prefill_attn(q, k, v, plan)
        torch.cuda.synchronize()
    finally:
        _lib.set_wait_limit(0, False)
    assert torch.isnan(out).all() and plan.status() == 1 and plan.status() == 0
    assert torch.equal(prefill.prefill_attn(q, k, v, plan), want)


def test_empty_batches(cuda):
    q, k, v = inputs([0, 0], [0, 7], 4, 2, 64)
    assert attend(cuda, q, k, v, [0, 0], [0, 7]).shape == (0, 4, 64)
    q, k, v = inputs([3], [0], 4, 2, 64)
    assert (attend(cuda, q, k, v, [3], [0]) == 0).all()


def test_out_must_not_overlap_the_inputs(cuda):
    from palu_b200 import prefill
    q, k, v = (t.to(cuda) for t in inputs([40], [40], 2, 2, 128))
    plan = prefill.PrefillPlan([40], n_q_heads=2, n_kv_heads=2, device=cuda)
    for out in (q, k, v):
        with pytest.raises(RuntimeError, match="overlap"):
            prefill.prefill_attn(q, k, v, plan, out=out)
    room = torch.empty(2, 40, 2, 128, dtype=torch.bfloat16, device=cuda)  # neighbours are fine
    room[0] = q
    assert torch.equal(prefill.prefill_attn(room[0], k, v, plan, out=room[1]), prefill.prefill_attn(q, k, v, plan))


def test_a_plan_made_on_another_stream(cuda):
    """The plan, and its token index, are used on a stream other than the one they were made on and then dropped."""
    from palu_b200 import prefill
    q, k, v = (t.to(cuda) for t in inputs([300, 7], [300, 90], 4, 2, 64))
    side = torch.cuda.Stream()
    plan = prefill.PrefillPlan([300, 7], [300, 90], rows=[3, 1], n_q_heads=4, n_kv_heads=2, device=cuda)
    want = prefill.prefill_attn(q, k, v, plan)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        rows, pos = plan.token_index()
        got = prefill.prefill_attn(q, k, v, plan)
        where = torch.stack([rows, pos])
        del plan, rows, pos
    full = torch.full((1 << 16,), -1, dtype=torch.int32, device=cuda)     # reuses the freed memory where it may
    torch.cuda.synchronize()
    assert torch.equal(got, want) and int(full.max()) == -1
    assert torch.equal(where.cpu(), torch.stack([torch.tensor([3] * 300 + [1] * 7), torch.tensor([*range(300), *range(83, 90)])]))


def test_token_index_is_not_laid_out_in_a_capture(cuda):
    from palu_b200 import prefill
    plan = prefill.PrefillPlan([3], n_q_heads=4, n_kv_heads=2, device=cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.zeros(1, device=cuda)
        with pytest.raises(RuntimeError, match="before capturing"):
            plan.token_index()


@pytest.mark.parametrize("d_v", [64, 128])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_a_reference_that_moves_among_large_scores(cuda, d_v, sign):
    """Scores of about +-2^20 that are exact integers (their tolerance is that of small ones: only differences matter). Eight
    tiles whose maxima stay within reach of the first reference, then a score that moves it: both parts weigh about the same,
    and an error of their relative weight by x would move the result by x / 2. The offset is the one at which the two references'
    products with log2 e, rounded to fp32, differ most."""
    import numpy as np
    log2e = np.float32(math.log2(math.e))
    slip = lambda m: float(np.float32(m) * log2e) - float(m) * float(log2e)
    base = int(sign) * 2**20
    e = max(range(200), key=lambda e: abs(slip(base + e) - slip(base + e + 13)))
    assert abs(slip(base + e) - slip(base + e + 13)) > 2.0 ** -4           # a weight off by 4 % if it entered the result
    n, rows = 9 * 128, 2
    offset = torch.full((n,), 6.0)
    offset[:32] = 0
    offset[1024:] = 0
    offset[1024] = 13
    q = torch.zeros(rows, 4, H)
    q[..., 0], q[..., 1] = 1024 * sign, 1.0
    k = torch.zeros(n, 1, H)
    k[..., 0], k[..., 1] = 1024.0, (offset + e)[:, None]
    v = torch.ones(n, 1, d_v)
    v[1024:] = -1
    q, k, v = (t.to(torch.bfloat16) for t in (q, k, v))
    assert float((offset + e).max()) <= 256                                 # integers that bf16 holds
    check(attend(cuda, q, k, v, [rows], [n], scale=1.0), q, k, v, [rows], [n], scale=1.0)


def _many_short(n):
    g = torch.Generator().manual_seed(20)
    q = torch.randint(1, 41, (n,), generator=g).tolist()
    return q, [x + (37 if i % 7 == 3 else 0) for i, x in enumerate(q)]


@pytest.mark.parametrize("d_v", [48, 64, 80, 128])
@pytest.mark.parametrize("batch", ["whole", "few_records", "many_records", "many_short"])
def test_non_finite_values_in_every_layout_of_the_work(cuda, d_v, batch):
    """Infinities and NaNs among the values, in the first and the last column: items that are whole, cut along the keys into
    few and into many records, and some hundreds of short prompts one after another on a thread block. A query that sees such
    a value gets it (of both signs, or a NaN: NaN), every other result keeps its bits."""
    from palu_b200 import prefill
    q_lens, k_lens = {"whole": ([90, 5, 300], [90, 5, 300]), "few_records": ([512], [2000]), "many_records": ([20], [6000]),
                      "many_short": _many_short(700)}[batch]
    plan = prefill.PrefillPlan(q_lens, k_lens, n_q_heads=8, n_kv_heads=2, device=cuda).info
    assert {"few_records": 0 < plan.n_merges * 2 <= plan.n_slots < 8 * plan.n_merges, "many_records": 0 < 8 * plan.n_merges <= plan.n_slots,
            "many_short": plan.n_merges == 0 and plan.n_pieces >= 4 * plan.n_ctas}.get(batch, plan.n_merges == 0)
    q, k, v = inputs(q_lens, k_lens, 8, 2, d_v, seed=21)
    bad, q0, k0 = [], 0, 0                                    # (first query row, its end, key row, KV head, column, value)
    for s, (ql, kl) in enumerate(zip(q_lens, k_lens)):
        if batch != "many_short" or s % 5 == 0:
            for i, h, x, y in ((ql // 3, 0, 0, math.inf), (ql // 2, 0, 0, -math.inf), (ql // 2, 1, d_v - 1, math.nan),
                               (ql - 1, 0, d_v - 1, math.inf)):
                bad.append((q0 + i, q0 + ql, k0 + kl - ql + i, h, x, y))
        q0, k0 = q0 + ql, k0 + kl
    v2 = v.clone()
    for b in bad:
        v2[b[2], b[3], b[4]] = b[5]
    clean = attend(cuda, q, k, v, q_lens, k_lens).float().cpu()
    got = attend(cuda, q, k, v2, q_lens, k_lens).float().cpu()
    want = clean.clone()
    for b in bad:
        want[b[0]:b[1], 4 * b[3]:4 * b[3] + 4, b[4]] += v2[b[2], b[3], b[4]].float()
    assert torch.equal(torch.nan_to_num(got, nan=7e30, posinf=8e30, neginf=9e30), torch.nan_to_num(want, nan=7e30, posinf=8e30, neginf=9e30))
