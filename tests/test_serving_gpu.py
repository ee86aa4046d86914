"""The packed prefill, the page pool and the scores together, through the layer and the decoder.

Tolerances. Against the fp32 path (``forward_prefill``, ``prefill_logits``) the packed path rounds q, K, V, the
probabilities and the result to bf16: five independent roundings of at most 2^-8 each, relative to sums whose errors average
like their terms, so a relative L2 error of at most 5 * 2^-8 = 2 % per layer; a decoder of two layers adds them, and its
random norm-preserving weights carry them to the logits: 4 %. What reads the same latents through other pages, or after a
fork or a compaction, is equal bit for bit.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

LAYER, DECODER = 5 * 2.0 ** -8, 10 * 2.0 ** -8


def rel_l2(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return ((a - b).norm() / b.norm()).item()


def make_layer(cuda, group, paged, max_seq=300, proj=torch.float32):
    from palu_b200.attention import PagedAttentionConfig, PaluAttention
    from palu_b200.convert import LowRank
    g = torch.Generator().manual_seed(1)
    dim, nh, nkv, r_k, r_v = 256, 8, 4, 64, 48
    VT = lambda r: torch.randn(nkv // group, r, dim, generator=g).repeat_interleave(group, 0) * dim ** -0.5
    U = lambda r: torch.randn(nkv, 128, r, generator=g) * r ** -0.5
    lr = LowRank(k_VT=VT(r_k), k_U=U(r_k), v_VT=VT(r_v), v_U=U(r_v), group_size=group)
    wq, wo = torch.randn(nh * 128, dim, generator=g) * dim ** -0.5, torch.randn(dim, nh * 128, generator=g) * (nh * 128) ** -0.5
    cfg = PagedAttentionConfig(block_size=16, max_num_blocks=80) if paged else None
    return PaluAttention(wq, wo, lr, nh, nkv, max_batch=4, max_seq=max_seq, device=cuda, paged_attention_config=cfg, proj_dtype=proj)


@pytest.mark.parametrize("paged", [False, True], ids=["contiguous", "paged"])
@pytest.mark.parametrize("group", [1, 2], ids=["per_head", "grouped"])
def test_packed_layer_against_the_padded_one(cuda, group, paged):
    from palu_b200 import prefill
    lens, rows = [70, 1, 129], [2, 0, 3]
    g = torch.Generator().manual_seed(2)
    xs = [torch.randn(n, 256, generator=g) for n in lens]
    plain = make_layer(cuda, group, False)
    want = torch.cat([plain.forward_prefill(x[None].to(cuda), user_id=r)[0] for x, r in zip(xs, rows)])
    layer = make_layer(cuda, group, paged)
    pt = None
    if paged:
        pt = torch.randperm(80, generator=g)[:4 * 19].view(4, 19).to(cuda, torch.int32)
    plan = prefill.PrefillPlan(lens, rows=rows, n_q_heads=8, n_kv_heads=4, device=cuda)
    got = layer.forward_prefill_packed(torch.cat(xs).to(cuda), plan, pt)
    assert rel_l2(got, want) <= LAYER
    if not paged:
        assert torch.equal(layer.k_cache, plain.k_cache) and torch.equal(layer.v_cache, plain.v_cache)
    # the prompts again in two chunks each (the second one behind its cached prefix): the same caches, the same result
    cut = [30, 0, 128]
    chunked = make_layer(cuda, group, paged)
    a = chunked.forward_prefill_packed(torch.cat([x[:c] for x, c in zip(xs, cut)]).to(cuda),
                                       prefill.PrefillPlan(cut, rows=rows, n_q_heads=8, n_kv_heads=4, device=cuda), pt)
    rest = [n - c for n, c in zip(lens, cut)]
    b = chunked.forward_prefill_packed(torch.cat([x[c:] for x, c in zip(xs, cut)]).to(cuda),
                                       prefill.PrefillPlan(rest, lens, rows=rows, n_q_heads=8, n_kv_heads=4, device=cuda), pt)
    parts = [torch.cat([p, q]) for p, q in zip(a.split(cut), b.split(rest))]
    assert rel_l2(torch.cat(parts), want) <= LAYER


def test_packed_layer_refusals(cuda):
    from palu_b200 import prefill
    layer = make_layer(cuda, 1, False)
    plan = lambda q, k=None, rows=None, nh=8: prefill.PrefillPlan(q, k, rows=rows, n_q_heads=nh, n_kv_heads=4, device=cuda)
    x = torch.zeros(5, 256, device=cuda)
    for needle, p in (("heads", plan([5], nh=16)), ("x must be", plan([4])), ("among its keys", plan([5], [4])),
                      ("among its keys", plan([5], [301])), ("distinct and below", plan([5], rows=[4])),
                      ("distinct and below", plan([3, 2], rows=[1, 1]))):
        with pytest.raises(RuntimeError, match=needle):
            layer.forward_prefill_packed(x, p)
    with pytest.raises(RuntimeError, match="page_table"):
        layer.forward_prefill_packed(x, plan([5]), torch.zeros(4, 19, dtype=torch.int32))


def make_decoder(cuda, paged, dtype=torch.float32):
    from palu_b200.attention import PagedAttentionConfig
    from palu_b200.model import DecoderConfig, PaluDecoder
    cfg = DecoderConfig(dim=512, n_layers=2, n_heads=4, n_kv_heads=2, ffn_dim=768, vocab=301)
    pc = PagedAttentionConfig(block_size=16, max_num_blocks=60) if paged else None
    return PaluDecoder(cfg, [(32, 64), (48, 32)], max_batch=6, max_seq=160, seed=5, device=cuda, proj_dtype=dtype, paged_attention_config=pc)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_serving_a_batch_with_shared_prefixes(cuda, dtype):
    """Admit three prompts, prefill them packed, fork one of them, decode all, finish one, compact, and decode on: every step
    against a decoder with contiguous caches that was given the same tokens row by row."""
    lens = [40, 17, 64]
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(301, (n,), generator=g) for n in lens]
    ref = make_decoder(cuda, False, dtype)
    m = make_decoder(cuda, True, dtype)
    pool = m.page_pool(6)
    pool.reserve([0, 1, 2], lens)
    logits = m.prefill_packed_logits(torch.cat(prompts), m.prefill_plan(lens), pool.table)
    want = torch.cat([ref.prefill_logits(p[None], row0=i) for i, p in enumerate(prompts)])
    assert rel_l2(logits, want) <= DECODER
    # rows 3 and 4 go on from row 0 and from the first 50 tokens of row 2; the reference takes its latents over
    pool.fork([0, 2], [3, 4], [40, 50])
    packed = make_decoder(cuda, False, dtype)              # contiguous caches filled by the packed path: the same latents
    packed.prefill_packed(torch.cat(prompts), packed.prefill_plan(lens))
    for L in packed.layers:
        for c in (L["attn"].k_cache, L["attn"].v_cache):
            c[3], c[4] = c[0], c[2]
    pos = torch.tensor([40, 17, 64, 40, 50, -1], dtype=torch.int32, device=cuda)
    for step in range(20):
        tok = torch.randint(301, (6,), generator=g).to(cuda)
        if step == 9:                                      # row 1 is finished; its pages are free, the others move together
            pool.free([1])
            pool.compact()
            pos[1] = -1
        live = [r for r in range(5) if not (step >= 9 and r == 1)]
        pool.reserve(live, [int(p) + 1 for p in pos[live]])
        a, b = m.decode_logits(tok, pos, pool.table), packed.decode_logits(tok, pos)
        assert torch.equal(a[live], b[live]), step
        pos[pos >= 0] += 1
    pool.check()
    used = int((pool.refs > 0).sum())
    assert int(pool.table.max()) < used + 5 * 2            # compacted at step 9; at most two pages a row since


def test_scores_of_a_packed_batch(cuda):
    lens = [33, 1, 0, 50]
    g = torch.Generator().manual_seed(4)
    tokens = torch.randint(301, (sum(lens),), generator=g)
    m = make_decoder(cuda, False)
    got = m.score(tokens, m.prefill_plan(lens), top=3, chunk=40)
    x = make_decoder(cuda, False).prefill_packed(tokens, m.prefill_plan(lens))
    logp = torch.log_softmax((x @ m.lm_head.t()).double(), -1).cpu()
    at = 0
    for n in lens:
        for i in range(n):
            t = at + i
            want = logp[t, tokens[t + 1]].item() if i + 1 < n else 0.0
            assert abs(got.logprob[t].item() - want) <= 1e-4 and abs(got.entropy[t].item() + (logp[t].exp() * logp[t]).sum().item()) <= 1e-4
        at += n
    assert torch.equal(got.top_id.cpu(), logp.topk(3, -1).indices)
    # and against the fp32 prefill: the log probability of a prompt's last step
    other = make_decoder(cuda, False)
    last = torch.log_softmax(other.prefill_logits(tokens[:32][None]).double(), -1)[0, tokens[32]].item()
    assert abs(got.logprob[31].item() - last) <= 0.1


def test_decode_logprobs(cuda):
    m = make_decoder(cuda, False)
    g = torch.Generator().manual_seed(5)
    prompt = torch.randint(301, (2, 12), generator=g)
    m.prefill_logits(prompt)
    tok, pos = torch.tensor([3, 4], device=cuda), torch.full((2,), 12, dtype=torch.int32, device=cuda)
    nxt, lp = m.decode_logprobs(tok, pos, top=2)
    logits = m.decode_logits(tok, pos)                      # the same latents at the same position again
    assert torch.equal(nxt, logits.argmax(-1)) and torch.equal(lp.top_id[:, 0], nxt) and torch.equal(lp.top_logprob[:, 0], lp.logprob)
    want = torch.log_softmax(logits.double(), -1)
    assert (lp.logprob.double() - want.gather(1, nxt[:, None])[:, 0]).abs().max() <= 1e-5


def test_page_pool_needs_paged_caches(cuda):
    with pytest.raises(RuntimeError, match="paged"):
        make_decoder(cuda, False).page_pool(2)


def test_a_batch_without_tokens(cuda):
    m = make_decoder(cuda, False)
    none, plan = torch.zeros(0, dtype=torch.long), m.prefill_plan([0, 0])
    assert m.prefill_packed(none, plan).shape == (0, 512) and m.prefill_packed_logits(none, plan).shape == (0, 301)
    got = m.score(none, plan, top=2)
    assert got.logprob.shape == (0,) and got.top_id.shape == (0, 2)
