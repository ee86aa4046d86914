"""Packed keys and values of cached latents on the GPU (palu_rebuild_kv) against the formula in 64 bits.

Tolerance per element, u = 2^-24: the sums over r products accumulate in fp32 (at most r additions: r u S, S the sum of
the products' absolute values), the rotation adds three roundings (4 u S), and the result is rounded to bf16 once
(2^-8 of it)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def tables(n):
    f = 500000.0 ** (-torch.arange(0, 128, 2).double() / 128)
    a = torch.arange(n).double()[:, None] * f
    return a.cos().float().repeat_interleave(2, -1).contiguous(), a.sin().float().repeat_interleave(2, -1).contiguous()


def make(lens, rows, n_kv, group, r_k, r_v, absorbed, seed=0):
    g = torch.Generator().manual_seed(seed)
    B, S, G = max(rows) + 1, max(max(lens), 1), n_kv // group
    k, v = torch.randn(B, G, S, r_k, generator=g).to(BF), torch.randn(B, G, S, r_v, generator=g).to(BF)
    u_k = (torch.randn(n_kv, r_k, 128, generator=g) * r_k ** -0.5).to(BF)
    u_v = None if absorbed else (torch.randn(n_kv, r_v, 128, generator=g) * r_v ** -0.5).to(BF)
    return k, v, u_k, u_v


def paged(cache, lens, rows, bs, n_blocks, g, width):
    """The cache's rows as pages in random places, and their table (-1 behind each row's pages)."""
    B, G, S, r = cache[0].shape[0], *cache[0].shape[1:3], None
    table = torch.full((B, width), -1, dtype=torch.int32)
    free = torch.randperm(n_blocks, generator=g).tolist()
    out = [torch.randn(n_blocks, G, bs, c.shape[3], generator=g).to(BF) for c in cache]
    for n, row in zip(lens, rows):
        for j in range(-(-n // bs)):
            b = table[row, j] = free.pop()
            part = slice(j * bs, min((j + 1) * bs, S))
            for o, c in zip(out, cache):
                o[b, :, :part.stop - part.start] = c[row, :, part]
    return out, table


def check(got_k, got_v, k, v, u_k, u_v, lens, rows, cos, sin, group):
    at = 0
    for n, row in zip(lens, rows):
        for h in range(u_k.shape[0]):
            x, w = k[row, h // group, :n].double(), u_k[h].double()
            y, s = x @ w, x.abs() @ w.abs()
            c, sn = cos[:n].double(), sin[:n].double()
            want = y * c + torch.stack([-y[:, 1::2], y[:, 0::2]], -1).flatten(-2) * sn
            S = s * c.abs() + torch.stack([s[:, 1::2], s[:, 0::2]], -1).flatten(-2) * sn.abs()
            err = (got_k[at:at + n, h].double().cpu() - want).abs()
            assert (err <= 2.0 ** -8 * want.abs() + (u_k.shape[1] + 4) * 2.0 ** -24 * S).all()
            if u_v is not None:
                x, w = v[row, h // group, :n].double(), u_v[h].double()
                want, S = x @ w, x.abs() @ w.abs()
                err = (got_v[at:at + n, h].double().cpu() - want).abs()
                assert (err <= 2.0 ** -8 * want.abs() + (u_v.shape[1] + 4) * 2.0 ** -24 * S).all()
            else:
                assert torch.equal(got_v[at:at + n, h].cpu(), v[row, h, :n])
        at += n
    assert at == got_k.shape[0] == got_v.shape[0]


CASES = [
    # lens, rows, n_kv, group, r_k, r_v, absorbed
    ([1], [0], 1, 1, 16, 16, True),
    ([5, 64, 65], [0, 1, 2], 8, 1, 64, 64, True),
    ([130, 0, 63], [2, 0, 1], 8, 1, 48, 112, True),
    ([200], [0], 4, 1, 128, 32, False),
    ([70, 1], [1, 0], 8, 4, 256, 256, False),
    ([129], [0], 8, 2, 160, 96, False),
]


@pytest.mark.parametrize("page", [0, 16, 64, 128])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{'_'.join(map(str, c[0]))}-g{c[3]}-r{c[4]}_{c[5]}")
def test_matches_the_formula(cuda, case, page):
    from palu_b200 import prefill
    lens, rows, n_kv, group, r_k, r_v, absorbed = case
    k, v, u_k, u_v = make(lens, rows, n_kv, group, r_k, r_v, absorbed)
    cos, sin = tables(max(lens))
    plan = prefill.PrefillPlan([0] * len(lens), lens, n_q_heads=n_kv, n_kv_heads=n_kv, rows=rows, device=cuda)
    kw = {"u_v": None if u_v is None else u_v.to(cuda)}
    kc, vc = k, v
    if page:
        width = -(-k.shape[2] // page)
        (kc, vc), table = paged((k, v), lens, rows, page, width * len(lens) + 3, torch.Generator().manual_seed(7), width)
        kw["page_table"] = table.to(cuda)
    gk, gv = prefill.rebuild_kv(kc.to(cuda), vc.to(cuda), u_k.to(cuda), cos.to(cuda), sin.to(cuda), plan, **kw)
    torch.cuda.synchronize()
    check(gk, gv, k, v, u_k, u_v, lens, rows, cos, sin, group)


def test_pages_that_the_table_does_not_name_read_as_zero(cuda):
    from palu_b200 import prefill
    k, v, u_k, u_v = make([64], [0], 2, 1, 32, 32, False)
    cos, sin = tables(64)
    table = torch.tensor([[1, -1, 9, 0]], dtype=torch.int32)       # 4 pages of 16; 9 is past the cache
    pool = [c[0].view(2, 4, 16, 32).transpose(0, 1).contiguous() for c in (k, v)]
    plan = prefill.PrefillPlan([0], [64], n_q_heads=2, n_kv_heads=2, device=cuda)
    gk, gv = prefill.rebuild_kv(pool[0].to(cuda), pool[1].to(cuda), u_k.to(cuda), cos.to(cuda), sin.to(cuda), plan, u_v=u_v.to(cuda),
                                page_table=table.to(cuda))
    k2, v2 = torch.zeros_like(k), torch.zeros_like(v)
    k2[0, :, :16], v2[0, :, :16] = k[0, :, 16:32], v[0, :, 16:32]
    k2[0, :, 48:], v2[0, :, 48:] = k[0, :, :16], v[0, :, :16]
    check(gk, gv, k2, v2, u_k, u_v, [64], [0], cos, sin, 1)
    assert (gk[16:48] == 0).all() and (gv[16:48] == 0).all()


def test_refusals(cuda):
    from palu_b200 import prefill
    k, v, u_k, u_v = (x.to(cuda) if x is not None else None for x in make([40], [0], 4, 2, 32, 32, False))
    cos, sin = (t.to(cuda) for t in tables(40))
    plan = prefill.PrefillPlan([0], [40], n_q_heads=4, n_kv_heads=4, device=cuda)
    call = lambda **kw: prefill.rebuild_kv(kw.pop("k", k), kw.pop("v", v), kw.pop("u_k", u_k), kw.pop("cos", cos), sin,
                                           kw.pop("plan", plan), **{"u_v": u_v, **kw})
    for needle, kw in (("need u_v", dict(u_v=None)), ("u_k must be", dict(u_k=u_k[:2])), ("fp32", dict(cos=cos[:39])),
                       ("bf16", dict(k=k.float())), ("same leading dims", dict(v=v[:, :, :30])),
                       ("must fit", dict(plan=prefill.PrefillPlan([0], [40], n_q_heads=4, n_kv_heads=4, rows=[1], device=cuda))),
                       ("must fit", dict(k=k[:, :, :39].contiguous(), v=v[:, :, :39].contiguous())),
                       ("heads_per_group", dict(k=k[:, :1].expand(-1, 3, -1, -1), v=v[:, :1].expand(-1, 3, -1, -1)))):
        with pytest.raises(RuntimeError, match=needle):
            call(**kw)


@pytest.mark.parametrize("absorbed", [False, True])
def test_an_expired_wait_gives_nan_and_a_status(cuda, absorbed):
    from palu_b200 import _lib, prefill
    lens = [200, 1, 33]
    k, v, u_k, u_v = (x.to(cuda) if x is not None else None for x in make(lens, [0, 1, 2], 4, 1, 64, 32, absorbed))
    cos, sin = (t.to(cuda) for t in tables(200))
    plan = prefill.PrefillPlan([0] * 3, lens, n_q_heads=4, n_kv_heads=4, device=cuda)
    want = prefill.rebuild_kv(k, v, u_k, cos, sin, plan, u_v=u_v)
    _lib.set_wait_limit(2_000_000, True)                    # 2 ms; the producer loads no factors
    try:
        got = prefill.rebuild_kv(k, v, u_k, cos, sin, plan, u_v=u_v)
        torch.cuda.synchronize()
    finally:
        _lib.set_wait_limit(0, False)
    assert torch.isnan(got[0]).all() and (torch.equal(got[1], want[1]) if absorbed else torch.isnan(got[1]).all())
    assert plan.status() == 1 and plan.status() == 0
    assert all(torch.equal(a, b) for a, b in zip(prefill.rebuild_kv(k, v, u_k, cos, sin, plan, u_v=u_v), want))


@pytest.mark.parametrize("n,n_kv,absorbed", [(400, 2, False), (400, 1, True), (70, 8, True)])
def test_many_units_on_a_thread_block(cuda, n, n_kv, absorbed):
    """Several units one after another on every thread block, neighbours of the same positions among them, whose tokens are
    fewer or more than the unit's before."""
    from palu_b200 import prefill
    lens = [(1, 130, 64, 257, 128, 5, 300, 77, 200)[(4 * i + i // 5) % 9] for i in range(n)]
    rows = torch.randperm(n, generator=torch.Generator().manual_seed(3)).tolist()
    k, v, u_k, u_v = make(lens, rows, n_kv, 1, 16, 16, absorbed)
    cos, sin = tables(300)
    plan = prefill.PrefillPlan([0] * n, lens, n_q_heads=n_kv, n_kv_heads=n_kv, rows=rows, device=cuda)
    gk, gv = prefill.rebuild_kv(k.to(cuda), v.to(cuda), u_k.to(cuda), cos.to(cuda), sin.to(cuda), plan,
                                u_v=None if u_v is None else u_v.to(cuda))
    torch.cuda.synchronize()
    assert plan.status() == 0
    check(gk, gv, k, v, u_k, u_v, lens, rows, cos, sin, 1)
