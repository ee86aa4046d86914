"""Token log probabilities on the GPU (palu_token_logprobs) against the formula in 64 bits.

Tolerance (fp32 arithmetic, u = 2^-24; M the row's maximum, R the sum over the other elements): x - M is rounded once;
each exponential is good to 2^-21 of itself (argument and approximation, for arguments above -40; smaller ones are below
2^-24 of the sum); R is a sum of at most n additions in a row per thread and about 20 joins: (n + 20) u. So log Z is off
by at most E = (n + 20) u + 2^-21, a log probability by E + 2 u (|x - M| + |log p|), and the entropy, whose second term
is a sum of the same kind with terms |d| e^d, by 3 E (1 + H + log1p R). Ids are exact.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def formula(logits, tokens, top):
    x = logits.double().cpu()
    m = x.amax(-1, keepdim=True)
    logp = torch.log_softmax(x, -1)
    pos = tokens.cpu().long()
    lp = logp.gather(1, pos.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    ent = -torch.where(x == -math.inf, torch.zeros_like(x), logp.exp() * logp).sum(-1)
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]      # equal values: the lower id first
    return lp, ent, logp.gather(1, ids), ids, (x - m)


def run(cuda, logits, tokens, top):
    from palu_b200 import scoring
    got = scoring.token_logprobs(logits, tokens, top)
    torch.cuda.synchronize()
    return [t.cpu() for t in got]


def check(cuda, logits, tokens, top):
    lp, ent, tv, ti = run(cuda, logits, tokens, top)
    wlp, went, wtv, wti, d = formula(logits, tokens, top)
    n = -(-logits.shape[1] // 256) + 16
    E = (n + 20) * U + 2.0 ** -21
    finite = torch.isfinite(wlp)
    assert torch.equal(torch.isneginf(lp), torch.isneginf(wlp))
    err = (lp.double() - wlp).abs()[finite]
    assert (err <= E + 2 * U * 2 * wlp.abs()[finite]).all(), err.max()
    z = torch.logsumexp(d, -1)
    assert ((ent.double() - went).abs() <= 3 * E * (1 + went + z)).all()
    assert torch.equal(ti, wti)
    fin = torch.isfinite(wtv)
    assert torch.equal(torch.isneginf(tv), ~fin)
    assert ((tv.double() - wtv).abs()[fin] <= E + 4 * U * wtv.abs()[fin]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("n,vocab,top", [(1, 1, 1), (1, 7, 3), (3, 33, 32), (2, 1000, 5), (1, 128256, 20), (5, 32001, 32), (37, 4099, 1),
                                         (300, 2048, 0), (700, 1031, 4), (64, 70000, 2)])
def test_matches_the_formula(cuda, dtype, n, vocab, top):
    g = torch.Generator().manual_seed(n + vocab)
    logits = (torch.randn(n, vocab, generator=g) * 3).to(cuda, dtype)
    check(cuda, logits, torch.randint(vocab, (n,), generator=g).to(cuda), top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shift", [1, 3, 7])
def test_rows_of_any_alignment_and_stride(cuda, dtype, shift):
    """A slice of a wider tensor: rows that start anywhere, other values around them."""
    g = torch.Generator().manual_seed(shift)
    wide = (torch.randn(9, 3011, generator=g) * 3).to(cuda, dtype)
    wide[:, :shift] = 1000.0
    wide[:, shift + 2500:] = 1000.0
    check(cuda, wide[:, shift:shift + 2500], torch.randint(2500, (9,), generator=g).to(cuda, torch.int32), 8)
    check(cuda, wide[:, shift:shift + 2], torch.randint(2, (9,), generator=g).to(cuda), 2)


def test_transposed_logits(cuda):
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(500, 6, generator=g).to(cuda).t()
    check(cuda, logits, torch.arange(6).to(cuda), 3)


@pytest.mark.parametrize("vocab", [999, 50000])
def test_ties_go_to_the_lowest_id(cuda, vocab):
    logits = torch.zeros(4, vocab, dtype=torch.bfloat16, device=cuda)
    logits[1, ::3] = 2.0
    logits[2, vocab // 2:] = -0.0                     # -0 and +0 are equal
    logits[3] = -math.inf
    logits[3, [5, 17, vocab - 1]] = 1.0
    check(cuda, logits, torch.tensor([0, 3, vocab - 1, 17], device=cuda), 32)


@pytest.mark.parametrize("rising", [True, False])
def test_sorted_logits(cuda, rising):
    """Every element a new maximum, or every later one smaller; the best 32 side by side."""
    x = torch.linspace(-20, 20, 40000, device=cuda)
    check(cuda, (x if rising else x.flip(0)).expand(3, -1).contiguous(), torch.tensor([0, 39999, 5], device=cuda), 32)


def test_one_thread_holds_the_best(cuda):
    """The 32 best values all in chunks that one thread of the kernel owns."""
    logits = torch.randn(1, 100000, generator=torch.Generator().manual_seed(2)).to(cuda)
    for i in range(32):
        logits[0, (37 + 256 * (i // 4)) * 4 + i % 4] = 50.0 + (i * 7) % 32
    check(cuda, logits, torch.tensor([148], device=cuda), 32)


def test_a_sure_token_keeps_its_small_numbers(cuda):
    """log p = -R with R far below 2^-24: relative accuracy, not absolute."""
    logits = torch.zeros(2, 1000, device=cuda)
    logits[0, 123], logits[1, 7] = 40.0, 25.0
    lp, ent, tv, ti = run(cuda, logits, torch.tensor([123, 7], device=cuda), 1)
    for i, top in enumerate((40.0, 25.0)):
        R = 999 * math.exp(-top)
        assert lp[i] == tv[i, 0] and abs(lp[i].item() + math.log1p(R)) <= 1e-5 * R
        assert abs(ent[i].item() - (math.log1p(R) + top * R / (1 + R))) <= 1e-4 * R * top


def test_masked_tokens(cuda):
    g = torch.Generator().manual_seed(3)
    logits = torch.randn(6, 5000, generator=g).to(cuda)
    logits[:, torch.rand(5000, generator=g).to(cuda) < 0.99] = -math.inf
    logits[0] = -math.inf
    logits[0, 4321] = -3.0                            # one token left: log p = 0, entropy 0
    check(cuda, logits, torch.tensor([4321, 1, 2, 3, 4, 5], device=cuda), 10)


def test_rows_without_a_distribution(cuda):
    logits = torch.randn(4, 3000, generator=torch.Generator().manual_seed(4)).to(cuda)
    logits[0] = -math.inf
    logits[1, 2000] = math.nan
    logits[2, [10, 2999]] = math.inf
    lp, ent, tv, ti = run(cuda, logits, torch.tensor([1, 1, 1, 1], device=cuda), 3)
    for i in range(3):
        assert torch.isnan(lp[i]) and torch.isnan(ent[i]) and torch.isnan(tv[i]).all()
    assert ti[0].tolist() == [0, 1, 2] and ti[1, 0] == 2000 and ti[2, :2].tolist() == [10, 2999]
    assert torch.isfinite(lp[3]) and torch.isfinite(tv[3]).all()


def test_tokens_outside_the_vocabulary(cuda):
    logits = torch.randn(3, 100, generator=torch.Generator().manual_seed(5)).to(cuda)
    lp, *_ = run(cuda, logits, torch.tensor([-1, 100, 99], device=cuda), 0)
    assert lp[0] == 0 and torch.isnan(lp[1]) and torch.isfinite(lp[2])


def test_same_bits_alone_in_a_batch_on_a_stream_and_in_a_graph(cuda):
    from palu_b200 import scoring
    g = torch.Generator().manual_seed(6)
    logits = (torch.randn(9, 20000, generator=g) * 3).to(cuda, torch.bfloat16)
    tokens = torch.randint(20000, (9,), generator=g).to(cuda)
    want = scoring.token_logprobs(logits, tokens, 7)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = [scoring.token_logprobs(logits, tokens, 7) for _ in range(3)]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = scoring.token_logprobs(logits, tokens, 7)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    for got in [*other, out]:
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_no_rows(cuda):
    lp, ent, tv, ti = run(cuda, torch.zeros(0, 50, device=cuda), torch.zeros(0, dtype=torch.long, device=cuda), 2)
    assert lp.shape == (0,) and tv.shape == (0, 2) and ti.dtype == torch.int64


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("first", [0.0, -math.inf, -3.0, -3.0e38, -1.0e6, 7.0e5], ids=str)
def test_rows_that_start_low_or_far_out(cuda, dtype, first):
    """The first half of the row at one value (zero, masked, the type's lowest, beyond fp32's fine range), the rest a
    little above it in another; a row that is one value throughout is uniform."""
    logits = torch.full((3, 40000), first).to(cuda, dtype)
    base = logits[0, 0].float().item()
    step = 4.0 if abs(base) < 1e5 or math.isinf(base) else abs(base) / 64
    logits[0, 20001::7] = (base if math.isfinite(base) else 0.0) + step
    logits[1, 39999] = (base if math.isfinite(base) else 0.0) + 2 * step
    logits[2, 17] = base if math.isfinite(base) else 0.0
    check(cuda, logits, torch.tensor([20001, 39999, 17], device=cuda), 5)


def test_the_lowest_finite_value_as_a_mask(cuda):
    logits = torch.full((2, 30000), torch.finfo(torch.bfloat16).min, dtype=torch.bfloat16, device=cuda)
    logits[0, [100, 29999]] = torch.tensor([1.0, 2.0], dtype=torch.bfloat16, device=cuda)
    check(cuda, logits, torch.tensor([100, 5], device=cuda), 4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("vocab", [1, 2, 3, 5, 9, 17, 127, 129])
def test_short_rows_of_minus_infinities(cuda, dtype, vocab):
    """Rows without a whole 16-byte chunk among them: the ids are the lowest, there is no distribution."""
    from palu_b200 import scoring
    top = min(vocab, 32)
    wide = torch.full((5, vocab + 3), -math.inf, device=cuda).to(dtype)
    for logits in (wide[:, :vocab], wide[:, 3:]):
        lp, ent, tv, ti = scoring.token_logprobs(logits, torch.zeros(5, dtype=torch.long, device=cuda), top)
        assert torch.isnan(lp).all() and torch.isnan(ent).all() and torch.isnan(tv).all()
        assert torch.equal(ti.cpu(), torch.arange(top).expand(5, -1))


def test_many_equal_elements_at_the_border_of_the_top(cuda):
    """More candidates than the kernel holds at a time: the rounds of its slow look, at several cluster sizes."""
    for n, vocab in ((1, 128256), (200, 40003), (900, 3001)):
        logits = torch.full((n, vocab), 1.0, device=cuda)
        logits[:, vocab // 3] = 2.0
        logits[n // 2, :vocab // 2] = 0.5
        check(cuda, logits, torch.zeros(n, dtype=torch.long, device=cuda), 9)


def test_a_vocabulary_past_32_bits_is_refused(cuda):
    from palu_b200 import scoring
    logits = torch.zeros(1, 1, dtype=torch.bfloat16, device=cuda).expand(1, 2**31)
    with pytest.raises(RuntimeError, match="vocab"):
        scoring.token_logprobs(logits, torch.zeros(1, dtype=torch.long, device=cuda))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("vocab", [4000, 40000])
@pytest.mark.parametrize("base", [-16000.0, -16512.0, -30080.0, -65280.0, -100352.0, -499712.0, 30080.0, 499712.0], ids=str)
def test_rows_far_from_zero(cuda, dtype, vocab, base):
    """Rows where a step of bf16 is 64 to 2048: every argument of an exponential is one fma against a reference, off by 2^-24
    of the difference and not of the logits, so the tolerance stays. Low values first and the next higher step later, in
    every part of the row that a thread block may read (from 5000 elements on); both steps mixed; one value; one higher one."""
    g = torch.Generator().manual_seed(7)
    step = 2.0 ** (math.floor(math.log2(abs(base))) - 7)
    logits = torch.full((5, vocab), base)
    logits[0, torch.arange(vocab) % 5000 >= 3500] = base + step
    logits[1] += step / 2 + 3 * torch.randn(vocab, generator=g)
    logits[3, vocab - 1] = base + step
    logits[4] += 40 * torch.randn(vocab, generator=g)
    logits = logits.to(cuda, dtype)
    assert logits[0].unique().numel() == 2 and logits[1].unique().numel() >= 2
    check(cuda, logits, torch.tensor([3999, 1, 2, vocab - 1, 17], device=cuda), 5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("top", [1, 3, 32])
@pytest.mark.parametrize("n,vocab", [(6, 3000), (7, 128256), (330, 9001)])
def test_a_nan_anywhere_comes_first(cuda, dtype, top, n, vocab):
    """NaN at the row's first and last places and between them, alone, twice and in numbers, of either sign, with one and with
    eight thread blocks a row: the lowest of their ids come first, then the other logits in order."""
    logits = torch.randn(n, vocab, generator=torch.Generator().manual_seed(vocab + top)) * 3
    places = ([10], [vocab // 2], [vocab - 1], [0, vocab - 2], list(range(5, vocab, 61)), [])
    for i in range(n):
        logits[i, places[i % 6]] = math.nan if i % 4 < 2 else -math.nan
    lp, ent, tv, ti = run(cuda, logits.to(cuda, dtype), torch.full((n,), 3, device=cuda), top)
    bad = torch.tensor([bool(places[i % 6]) for i in range(n)])
    want = torch.sort(logits.to(dtype).double(), dim=-1, descending=True, stable=True).indices[:, :top]   # NaN is the largest
    assert (ti >= 0).all() and (ti < vocab).all() and torch.equal(ti, want)
    for t in (lp, ent, tv[:, 0]):
        assert torch.equal(torch.isnan(t), bad)
