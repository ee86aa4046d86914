"""Operators of serving a decoder with latent key-value caches: their cases, plain forms and exact values.

* prefill: causal attention of packed prompts (or prompt chunks behind a cached prefix) with grouped heads;
* rebuild: the packed, rotated keys and the values of cached latents, contiguous or paged;
* logprobs: log probabilities of given tokens with the entropy and the top alternatives;
* pages: copying, forking, freeing and compacting the pages of paged caches.

``own`` false: elementary torch operations, in 32 bits, rounded once at the end. ``own`` true: this repository's
operators. Shapes follow the decoder's configuration (32 query heads, 8 KV heads of 128, rank-64 latents, a
vocabulary of 128256, pages of 64 positions) unless a case says otherwise.
"""
import math
import sys
from pathlib import Path

import torch

own = False

HEAD = 128
_PACKAGE = str(Path(__file__).resolve().parents[1] / "tt-cadlab_b200")


def _own_modules():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from palu_b200 import paging, prefill, scoring
    return prefill, scoring, paging


def _ints(text):
    return [int(x) for x in text.split(",")]


def _text(values):
    return ",".join(str(int(v)) for v in values)


# ---- cases ------------------------------------------------------------------------------------------------

def listed():
    return [
        # short prompts arriving together, one of them a single token: launch and pipeline latency
        dict(name="prefill_short", op="prefill", q_lens="1,17,33,128", k_lens="1,17,33,128", n_q=32, n_kv=8, d_v=64),
        # an ordinary batch of prompts of different lengths (per-head latents: values stay rank 64)
        dict(name="prefill_ragged", op="prefill", q_lens="2048,511,1000,1777,64,129,900,1763",
             k_lens="2048,511,1000,1777,64,129,900,1763", n_q=32, n_kv=8, d_v=64),
        # two chunks of long prompts, each behind its cached prefix: few query rows, many keys
        dict(name="prefill_chunk", op="prefill", q_lens="256,499", k_lens="16384,9001", n_q=32, n_kv=8, d_v=128),
        # one long prompt (grouped latents: values rebuilt to the full head dim)
        dict(name="prefill_long", op="prefill", q_lens="32768", k_lens="32768", n_q=32, n_kv=8, d_v=128),
        # paged grouped latents of a few short rows before a prompt chunk
        dict(name="rebuild_paged", op="rebuild", lens="700,1,333,64,129", n_kv=8, group=4, r_k=256, r_v=256, page=64),
        # a full batch of per-head latents at the decode benchmark's size
        dict(name="rebuild_full", op="rebuild", lens=_text([8192] * 32), n_kv=8, group=1, r_k=64, r_v=64, page=0),
        # one decode step of one row, its log probability and five alternatives
        dict(name="logprobs_step", op="logprobs", n=1, vocab=128256, bits=16, top=5, masked=0.0),
        # a decode batch with a grammar mask over an odd vocabulary, fp32 logits, twenty alternatives
        dict(name="logprobs_batch", op="logprobs", n=129, vocab=32001, bits=32, top=20, masked=0.5),
        # scoring a packed prompt (perplexity): one row per token
        dict(name="logprobs_score", op="logprobs", n=4096, vocab=128256, bits=16, top=1, masked=0.0),
        # one request forked into four samples on a small model, and the samples freed again
        dict(name="pages_fork", op="fork", layers=2, heads=8, r_k=64, r_v=64, page=64, blocks=64, lens="777", children=4),
        # a batch forked in every layer of the decoder (beam steps), and freed again
        dict(name="pages_beam", op="fork", layers=32, heads=8, r_k=64, r_v=32, page=64, blocks=600,
             lens="1000,2047,64,515,1500,3000,129,4000", children=3),
        # a fragmented pool compacted in every layer of the decoder
        dict(name="pages_compact", op="compact", layers=32, heads=8, r_k=64, r_v=64, page=64, blocks=512, rows=12, per_row=24),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _pairs(q_lens, k_lens):
    """Visible (query, key) pairs of causal attention, the last query aligned with the last key."""
    total = 0
    for q, k in zip(q_lens, k_lens):
        first = k - q + 1                       # keys visible to the first query
        skip = max(0, -first + 1) if first < 1 else 0
        n = q - skip
        total += n * (max(first, 1) + k) // 2
    return total


_MOST_PAIRS = 32768 * 32769 // 2 * 32


def draw(rng):
    op = rng.choice(["prefill", "prefill", "rebuild", "logprobs", "logprobs", "fork", "compact"])
    if op == "prefill":
        n_kv, rep = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 4, 5, 8])
        while True:
            rows = _log(rng, 1, 24)
            q = [_log(rng, 1, 8192) for _ in range(rows)]
            k = [x + (_log(rng, 1, 16384) if rng.random() < 0.3 else 0) for x in q]
            if _pairs(q, k) * n_kv * rep <= _MOST_PAIRS and sum(q) <= 32768 and sum(k) <= 65536:
                break
        return dict(op=op, q_lens=_text(q), k_lens=_text(k), n_q=n_kv * rep, n_kv=n_kv, d_v=16 * rng.randint(1, 8))
    if op == "rebuild":
        group = rng.choice([1, 1, 2, 4])
        while True:
            lens = [_log(rng, 1, 16384) for _ in range(_log(rng, 1, 32))]
            if sum(lens) <= 131072:
                break
        r_k, r_v = (16 * rng.randint(1, 8), 16 * rng.randint(1, 8)) if group == 1 else (32 * rng.randint(1, 8), 32 * rng.randint(1, 8))
        return dict(op=op, lens=_text(lens), n_kv=8, group=group, r_k=r_k, r_v=r_v, page=rng.choice([0, 16, 32, 64, 128]))
    if op == "logprobs":
        while True:
            n, vocab = _log(rng, 1, 4096), _log(rng, 1000, 262144)
            if n * vocab <= 4096 * 128256:
                break
        return dict(op=op, n=n, vocab=vocab, bits=rng.choice([16, 16, 32]), top=rng.choice([0, 1, 5, 20, 32]),
                    masked=rng.choice([0.0, 0.0, 0.5, 0.999]))
    r_k, r_v, page, layers = rng.choice([32, 48, 64, 96, 128]), rng.choice([32, 48, 64, 96, 128]), rng.choice([16, 32, 64, 128]), _log(rng, 1, 32)
    blocks = max(40, min(2048, int(2.0e9 / (layers * 8 * page * (r_k + r_v) * 2))))
    if op == "fork":
        lens, room = [], blocks // 2
        for _ in range(_log(rng, 1, 16)):
            n = _log(rng, 1, 4096)
            if room - -(-n // page) - 4 < 0:
                break
            room -= -(-n // page) + 4
            lens.append(n)
        return dict(op=op, layers=layers, heads=8, r_k=r_k, r_v=r_v, page=page, blocks=blocks, lens=_text(lens or [5]),
                    children=rng.randint(1, 4))
    rows = rng.randint(1, 32)
    return dict(op="compact", layers=layers, heads=8, r_k=r_k, r_v=r_v, page=page, blocks=blocks, rows=rows,
                per_row=max(1, int(blocks * rng.uniform(0.2, 0.9) / rows)))


# ---- inputs -----------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _rope_tables(n):
    """cos and sin of n positions, [n, 128] fp32, each frequency twice side by side (theta 500000)."""
    f = 500000.0 ** (-torch.arange(0, HEAD, 2, dtype=torch.float64, device="cuda") / HEAD)
    ang = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * f
    return (torch.cos(ang).float().repeat_interleave(2, -1).contiguous(),
            torch.sin(ang).float().repeat_interleave(2, -1).contiguous())


def _prefill_inputs(case, seed):
    g, tq, tk = _gen(seed), sum(_ints(case["q_lens"])), sum(_ints(case["k_lens"]))
    return (_normal(g, tq, case["n_q"], HEAD), _normal(g, tk, case["n_kv"], HEAD), _normal(g, tk, case["n_kv"], case["d_v"]))


def _rebuild_inputs(case, seed):
    g, lens, page = _gen(seed), _ints(case["lens"]), case["page"]
    groups, longest = case["n_kv"] // case["group"], max(lens)
    if page:
        per_row = -(-longest // page)
        blocks = sum(-(-n // page) for n in lens) + 3
        order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
        used, at = torch.full((len(lens), per_row), -1, dtype=torch.int32, device="cuda"), 0
        for b, n in enumerate(lens):
            m = -(-n // page)
            used[b, :m] = order[at:at + m]
            at += m
        lead, table = (blocks, groups, page), used
    else:
        lead, table = (len(lens), groups, longest), None
    k, v = _normal(g, *lead, case["r_k"]), _normal(g, *lead, case["r_v"])
    u_k = _normal(g, case["n_kv"], case["r_k"], HEAD, scale=case["r_k"] ** -0.5)
    u_v = _normal(g, case["n_kv"], case["r_v"], HEAD, scale=case["r_v"] ** -0.5) if case["group"] > 1 else None
    cos, sin = _rope_tables(longest)
    return k, v, u_k, u_v, cos, sin, table


def _logprob_inputs(case, seed):
    g, n, vocab = _gen(seed), case["n"], case["vocab"]
    logits = torch.empty(n, vocab, dtype=torch.bfloat16 if case["bits"] == 16 else torch.float32, device="cuda")
    for a in range(0, n, 512):
        logits[a:a + 512] = torch.randn(min(512, n - a), vocab, generator=g, device="cuda") * 3.0
    tokens = torch.randint(vocab, (n,), generator=g, device="cuda")
    if case["masked"]:
        hide = torch.rand(vocab, generator=g, device="cuda") < case["masked"]
        hide[tokens[::2]] = False               # every other given token is one the mask allows
        logits[:, hide] = -math.inf
    return logits, tokens


def _flat_caches(case, seed):
    """Every layer's K and V cache [blocks, heads, page, r], views of one flat buffer."""
    shape = (case["blocks"], case["heads"], case["page"])
    per = math.prod(shape)
    flat = torch.empty(case["layers"] * per * (case["r_k"] + case["r_v"]), dtype=torch.bfloat16, device="cuda")
    flat.normal_(generator=_gen(seed))
    caches, at = [], 0
    for _ in range(case["layers"]):
        for r in (case["r_k"], case["r_v"]):
            caches.append(flat[at:at + per * r].view(*shape, r))
            at += per * r
    return flat, caches


def _page_inputs(case, seed):
    """Caches, and a page table [rows, entries] over pages in random order with its counts of pages and references."""
    flat, caches = _flat_caches(case, seed)
    gen = torch.Generator().manual_seed(int(seed))
    order = torch.randperm(case["blocks"], generator=gen).to(torch.int32)
    if case["op"] == "fork":
        counts = [-(-n // case["page"]) for n in _ints(case["lens"])]
        rows, width = len(counts) * (1 + case["children"]), max(counts)
    else:
        counts = [case["per_row"]] * case["rows"]
        rows, width = case["rows"] + 1, case["per_row"]
    table, mapped, at = torch.full((rows, width), -1, dtype=torch.int32), torch.zeros(rows, dtype=torch.int32), 0
    for b, m in enumerate(counts):
        table[b, :m] = order[at:at + m]
        mapped[b] = m
        at += m
    if case["op"] == "compact":                 # one more row shares the first row's pages, as a fork leaves it
        table[-1], mapped[-1] = table[0], mapped[0]
    refs = torch.zeros(case["blocks"], dtype=torch.int32)
    used = table[table >= 0].long()
    refs.index_add_(0, used, torch.ones(used.numel(), dtype=torch.int32))
    return flat, caches, table.cuda(), refs.cuda(), mapped.cuda()


def _fork_lists(case):
    lens, children = _ints(case["lens"]), case["children"]
    parents = [p for p in range(len(lens)) for _ in range(children)]
    kids = [len(lens) + i for i in range(len(parents))]
    return parents, kids, [lens[p] for p in parents]


def prepare(case, seed):
    op, state = case["op"], dict(case)
    if op == "prefill":
        state["q"], state["k"], state["v"] = _prefill_inputs(case, seed)
        if own:
            prefill, _, _ = _own_modules()
            state["plan"] = prefill.PrefillPlan(_ints(case["q_lens"]), _ints(case["k_lens"]), n_q_heads=case["n_q"], n_kv_heads=case["n_kv"])
            state["call"] = prefill.prefill_attn
    elif op == "rebuild":
        (state["k"], state["v"], state["u_k"], state["u_v"], state["cos"], state["sin"], state["table"]) = _rebuild_inputs(case, seed)
        state["lens"] = _ints(case["lens"])
        if own:
            prefill, _, _ = _own_modules()
            state["plan"] = prefill.PrefillPlan([0] * len(state["lens"]), state["lens"], n_q_heads=case["n_kv"], n_kv_heads=case["n_kv"])
            state["call"] = prefill.rebuild_kv
    elif op == "logprobs":
        state["logits"], state["tokens"] = _logprob_inputs(case, seed)
        if own:
            state["call"] = _own_modules()[1].token_logprobs
    else:
        state["flat"], state["caches"], table, refs, mapped = _page_inputs(case, seed)
        if op == "fork":
            state["lists"] = _fork_lists(case)
        if own:
            paging = _own_modules()[2]
            state["pool"] = pool = paging.PagePool(state["caches"], rows=table.shape[0], blocks_per_row=table.shape[1])
            pool.table.copy_(table)
            pool.refs.copy_(refs)
            pool.mapped.copy_(mapped)
            state["saved"] = pool.state.clone()
        else:
            state["table"], state["refs"], state["mapped"] = table, refs, mapped
    return state


# ---- one pass ---------------------------------------------------------------------------------------------

def run(state):
    op = state["op"]
    if op == "prefill":
        if own:
            return state["call"](state["q"], state["k"], state["v"], state["plan"])
        return _plain_prefill(state["q"], state["k"], state["v"], _ints(state["q_lens"]), _ints(state["k_lens"]))
    if op == "rebuild":
        if own:
            return state["call"](state["k"], state["v"], state["u_k"], state["cos"], state["sin"], state["plan"], u_v=state["u_v"],
                                 page_table=state["table"])
        return _plain_rebuild(state)
    if op == "logprobs":
        if own:
            return state["call"](state["logits"], state["tokens"], state["top"])
        return _plain_logprobs(state["logits"], state["tokens"], state["top"])
    if op == "fork":
        parents, kids, lens = state["lists"]
        if own:
            pool = state["pool"]
            pool.fork(parents, kids, lens)
            pool.free(kids)
            return state["flat"], pool.table, pool.refs, pool.mapped
        return _plain_fork(state, parents, kids, lens)
    if own:
        pool = state["pool"]
        pool.state.copy_(state["saved"])        # the fragmented pool again; the pages keep their contents
        pool.compact()
        return state["flat"], pool.table, pool.refs, pool.mapped
    return _plain_compact(state)


def _plain_prefill(q, k, v, q_lens, k_lens):
    n_kv, rep = k.shape[1], q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape[0], q.shape[1], v.shape[2], dtype=torch.float32, device=q.device)
    q0 = k0 = 0
    for ql, kl in zip(q_lens, k_lens):
        ks = k[k0:k0 + kl].float().permute(1, 2, 0)                                 # [n_kv, 128, kl]
        vs = v[k0:k0 + kl].float().transpose(0, 1)                                  # [n_kv, kl, d_v]
        step = max(1, (1 << 28) // (n_kv * rep * max(kl, 1)))
        for a in range(0, ql, step):
            n = min(step, ql - a)
            seen = min(max(kl - ql + a + n, 0), kl)                                  # keys that the last of these queries sees
            if seen == 0:
                continue
            qs = q[q0 + a:q0 + a + n].float().view(n, n_kv, rep, HEAD).permute(1, 0, 2, 3).reshape(n_kv, n * rep, HEAD)
            s = (qs @ ks[:, :, :seen] * HEAD ** -0.5).view(n_kv, n, rep, seen)
            last = torch.arange(a, a + n, device=q.device) + (kl - ql)               # the last key that each query sees
            hidden = torch.arange(seen, device=q.device)[None, :] > last[:, None]
            s = s.masked_fill(hidden[None, :, None, :], -math.inf)
            e = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
            total = e.sum(-1, keepdim=True)
            o = (e.view(n_kv, n * rep, seen) @ vs[:, :seen]).view(n_kv, n, rep, -1)
            o = torch.where(total > 0, o / total, torch.zeros_like(o))
            out[q0 + a:q0 + a + n] = o.permute(1, 0, 2, 3).reshape(n, n_kv * rep, -1)
        q0, k0 = q0 + ql, k0 + kl
    return out.to(torch.bfloat16)


def _gather_rows(cache, lens, table):
    """Cached latents of all rows one after another: [sum(lens), groups, r]."""
    dev = cache.device
    n = torch.tensor(lens, device=dev)
    row = torch.repeat_interleave(torch.arange(len(lens), device=dev), n)
    pos = torch.arange(row.numel(), device=dev) - torch.repeat_interleave(n.cumsum(0) - n, n)
    if table is None:
        return cache[row, :, pos], pos
    page = cache.shape[2]
    return cache[table[row, pos // page].long(), :, pos % page], pos


def _plain_rebuild(state):
    group = state["group"]
    lk, pos = _gather_rows(state["k"], state["lens"], state["table"])
    lv, _ = _gather_rows(state["v"], state["lens"], state["table"])
    k = torch.einsum("tgr,gdrh->tgdh", lk.float(), state["u_k"].float().view(-1, group, state["r_k"], HEAD)).reshape(lk.shape[0], -1, HEAD)
    c, s = state["cos"][pos][:, None], state["sin"][pos][:, None]
    k = k * c + torch.stack([-k[..., 1::2], k[..., 0::2]], -1).flatten(-2) * s
    if state["u_v"] is None:
        return k.to(torch.bfloat16), lv
    v = torch.einsum("tgr,gdrh->tgdh", lv.float(), state["u_v"].float().view(-1, group, state["r_v"], HEAD)).reshape(lv.shape[0], -1, HEAD)
    return k.to(torch.bfloat16), v.to(torch.bfloat16)


def _plain_logprobs(logits, tokens, top):
    n, vocab = logits.shape
    lp, ent = torch.empty(n, device=logits.device), torch.empty(n, device=logits.device)
    tv = torch.empty(n, top, device=logits.device)
    ti = torch.empty(n, top, dtype=torch.int64, device=logits.device)
    back = vocab - 1 - torch.arange(vocab, device=logits.device)
    step = max(1, (1 << 27) // vocab)
    for a in range(0, n, step):
        x = logits[a:a + step].float()
        d = x - x.amax(-1, keepdim=True)
        e = torch.exp(d)
        total = e.sum(-1)
        log_total = torch.log(total)
        lp[a:a + step] = d.gather(1, tokens[a:a + step, None])[:, 0] - log_total
        ent[a:a + step] = log_total - torch.where(e > 0, e * d, torch.zeros_like(d)).sum(-1) / total
        if top:
            # order by value, then by the lower index: one whole number that holds both
            b = (x + 0.0).view(torch.int32).long()
            best = (torch.where(b < 0, -(b & 0x7FFFFFFF), b) * (1 << 20) + back).topk(top, -1).values
            ti[a:a + step] = vocab - 1 - (best & ((1 << 20) - 1))
            tv[a:a + step] = d.gather(1, ti[a:a + step]) - log_total[:, None]
    return lp, ent, tv, ti


def _plain_fork(state, parents, kids, lens):
    page, dev = state["page"], state["flat"].device
    table, refs, mapped = state["table"].clone(), state["refs"].clone(), state["mapped"].clone()
    parents, kids, n = (torch.tensor(x, device=dev) for x in (parents, kids, lens))
    full, count = n // page, -(-n // page)
    j = torch.arange(table.shape[1], device=dev)[None]
    child = torch.where(j < full[:, None], table[parents], torch.full_like(table[parents], -1))
    part = count > full
    rank = part.long().cumsum(0) - 1
    free = torch.argsort((refs != 0).to(torch.int8), stable=True)                     # free pages, lowest first
    new = torch.where(part, free[rank.clamp(min=0)], -torch.ones_like(rank))
    child = torch.where((j == full[:, None]) & part[:, None], new[:, None].to(torch.int32), child)
    old = table[parents, full.clamp(max=table.shape[1] - 1)].long()
    src, dst = old[part], new[part]
    for c in state["caches"]:
        c[dst] = c[src]
    table[kids] = child
    mapped[kids] = count.to(torch.int32)
    taken = child[child >= 0].long()
    one = torch.ones_like(taken, dtype=torch.int32)
    refs.index_add_(0, taken, one)
    refs.index_add_(0, taken, -one)                                                  # and the children freed again
    table[kids] = -1
    mapped[kids] = 0
    return state["flat"], table, refs, mapped


def _plain_compact(state):
    refs = state["refs"]
    live = refs > 0
    count = live.sum()
    at = torch.arange(refs.numel(), device=refs.device)
    src, dst = at[live & (at >= count)], at[~live & (at < count)]                    # moves, lowest page to lowest hole
    for c in state["caches"]:
        c[dst] = c[src]
    to = at.clone()
    to[src] = dst
    moved = refs.clone()
    moved[dst] = refs[src]
    moved[src] = 0
    table = state["table"]
    return state["flat"], torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), table), moved, state["mapped"].clone()


# ---- work -------------------------------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "prefill":
        q, k = _ints(case["q_lens"]), _ints(case["k_lens"])
        read = sum(q) * case["n_q"] * HEAD + sum(k) * case["n_kv"] * (HEAD + case["d_v"])
        return {"bytes": 2 * (read + sum(q) * case["n_q"] * case["d_v"]), "flops": 2 * _pairs(q, k) * case["n_q"] * (HEAD + case["d_v"])}
    if op == "rebuild":
        t, n_kv, groups = sum(_ints(case["lens"])), case["n_kv"], case["n_kv"] // case["group"]
        r_k, r_v = case["r_k"], case["r_v"]
        u = n_kv * HEAD * (r_k + (r_v if case["group"] > 1 else 0))
        out = n_kv * HEAD + (n_kv * HEAD if case["group"] > 1 else groups * r_v)
        tables = 4 * max(_ints(case["lens"])) * HEAD                                  # each frequency's cos and sin once
        flops = 2 * t * n_kv * HEAD * (r_k + (r_v if case["group"] > 1 else 0)) + 3 * t * n_kv * HEAD
        return {"bytes": 2 * (t * groups * (r_k + r_v) + u + t * out) + tables, "flops": flops}
    if op == "logprobs":
        n, vocab = case["n"], case["vocab"]
        return {"bytes": n * vocab * case["bits"] // 8 + n * (8 + 8 + 12 * case["top"]), "flops": 6 * n * vocab}
    page_bytes = case["layers"] * case["heads"] * case["page"] * (case["r_k"] + case["r_v"]) * 2
    if op == "fork":
        _, _, lens = _fork_lists(case)
        pages = sum(1 for n in lens if n % case["page"])
        entries = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": 2 * pages * page_bytes + 4 * (case["blocks"] + 6 * entries), "flops": 0}
    live = min(case["blocks"], case["rows"] * case["per_row"])
    moved = live * (case["blocks"] - live) // case["blocks"]                         # expected for pages in random places
    return {"bytes": 2 * moved * page_bytes + 8 * (case["blocks"] + (case["rows"] + 1) * case["per_row"]), "flops": 0}


# ---- exact values -----------------------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "prefill":
        return _exact_prefill(case, seed)
    if case["op"] == "rebuild":
        return _exact_rebuild(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(case, seed)
    return None                                  # pages are moved, not computed


def _exact_prefill(case, seed):
    q, k, v = _prefill_inputs(case, seed)
    rep = case["n_q"] // case["n_kv"]
    q_lens, k_lens = _ints(case["q_lens"]), _ints(case["k_lens"])
    out = torch.zeros(q.shape[0], case["n_q"], case["d_v"], dtype=torch.float64, device=q.device)
    for h in range(case["n_q"]):
        q0 = k0 = 0
        for ql, kl in zip(q_lens, k_lens):
            ks, vs = k[k0:k0 + kl, h // rep].double(), v[k0:k0 + kl, h // rep].double()
            for a in range(0, ql, 4096):
                b = min(ql, a + 4096)
                n = max(0, kl - ql + b)          # keys up to the last query's own
                if n:
                    s = q[q0 + a:q0 + b, h].double() @ ks[:n].T / math.sqrt(HEAD)
                    # query a + i sees keys 0 .. kl - ql + a + i
                    see = torch.ones(b - a, n, dtype=torch.bool, device=q.device).tril(kl - ql + a)
                    p = torch.softmax(s.masked_fill(~see, -math.inf), -1)
                    out[q0 + a:q0 + b, h] = torch.nan_to_num(p) @ vs[:n]
            q0, k0 = q0 + ql, k0 + kl
    return out


def _exact_rebuild(case, seed):
    k, v, u_k, u_v, cos, sin, table = _rebuild_inputs(case, seed)
    lens, heads, page = _ints(case["lens"]), case["n_kv"], case["page"]
    keys = torch.empty(sum(lens), heads, HEAD, dtype=torch.float64, device=k.device)
    values = torch.empty(sum(lens), heads, HEAD if u_v is not None else case["r_v"], dtype=torch.float64, device=k.device)
    at = 0
    for b, n in enumerate(lens):
        def row(cache, g):
            if table is None:
                return cache[b, g, :n].double()
            return torch.cat([cache[i, g] for i in table[b, :-(-n // page)].tolist()])[:n].double()
        z = torch.complex(cos[:n, ::2].double(), sin[:n, ::2].double())
        for h in range(heads):
            g = h // case["group"]
            x = row(k, g) @ u_k[h].double()
            keys[at:at + n, h] = torch.view_as_real(torch.complex(x[:, ::2].contiguous(), x[:, 1::2].contiguous()) * z).flatten(-2)
            values[at:at + n, h] = row(v, g) @ u_v[h].double() if u_v is not None else row(v, g)
        at += n
    return keys, values


def _exact_logprobs(case, seed):
    logits, tokens = _logprob_inputs(case, seed)
    lp, ent, tv, ti = [], [], [], []
    for a in range(0, case["n"], 256):
        x = logits[a:a + 256].double()
        logp = torch.log_softmax(x, -1)
        lp.append(logp.gather(1, tokens[a:a + 256, None])[:, 0])
        ent.append(-(logp.exp() * logp.clamp(min=-1e300)).sum(-1))
        if case["top"]:
            # a stable descending sort leaves the lower index first among equals; only the first entries can matter
            cut = x.topk(case["top"], -1).values[:, -1:]
            at = torch.arange(case["vocab"], device=x.device).expand_as(x)
            over, tie = x > cut, x == cut
            keep = over | (tie & (tie.long().cumsum(-1) <= case["top"] - over.sum(-1, keepdim=True)))
            ids = at[keep].view(x.shape[0], case["top"])
            order = torch.sort(x.gather(1, ids), dim=-1, descending=True, stable=True).indices
            ids = ids.gather(1, order)
            ti.append(ids)
            tv.append(logp.gather(1, ids))
    n = case["n"]
    empty = torch.empty(n, 0, dtype=torch.float64, device=logits.device)
    return (torch.cat(lp), torch.cat(ent), torch.cat(tv) if tv else empty, torch.cat(ti) if ti else empty.long())
