"""Prefill of packed prompts: the batch's plan, the causal attention over it, and the keys and values of a cached prefix.

A packed batch holds sequences of different lengths one after another, without padding: sequence s has ``q_lens[s]``
query positions and ``k_lens[s]`` keys, its last query aligned with its last key (a prompt: equal lengths; a prompt
chunk behind a cached prefix: more keys than queries). ``PrefillPlan`` lays the batch's work out once, on the host;
every layer of a forward pass then uses it (``rebuild_kv``, ``prefill_attn``). The reference prefills one user's padded prompt at a
time with the stock attention op (palu_tt/attention.py:382-516).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from palu_b200 import _lib

HEAD_DIM = 128
_SCALE = HEAD_DIM ** -0.5


def _lengths(x, what: str):
    """Host lengths (a sequence or an integer CPU tensor) as a ctypes int32 array."""
    if isinstance(x, torch.Tensor):
        if x.is_cuda:
            raise RuntimeError(f"{what} must be on the host (a sequence or a CPU tensor): the plan is laid out there")
        x = x.reshape(-1).tolist()
    x = [int(v) for v in x]
    if any(not -2**31 <= v < 2**31 for v in x):
        raise RuntimeError(f"{what} must fit 32 bits")
    return (ctypes.c_int32 * len(x))(*x), x


class PrefillPlan:
    """The work of one packed batch, laid out for the GPU (palu_plan_prefill).

    ``q_lens`` / ``k_lens``: host lengths per sequence (``k_lens`` None: equal to ``q_lens``). ``rows``: the cache row of
    each sequence, for ``rebuild_kv`` (None: 0, 1, ...). Building a plan copies it to ``device`` and waits for the copy, so
    build it outside a CUDA graph capture; it can then be used on any stream of that device, by any number of calls, also
    at the same time. Keep it as long as a captured graph that uses it."""

    def __init__(self, q_lens: Sequence[int], k_lens: Optional[Sequence[int]] = None, *, n_q_heads: int, n_kv_heads: int,
                 rows: Optional[Sequence[int]] = None, device="cuda"):
        ql, self.q_lens = _lengths(q_lens, "q_lens")
        kl, self.k_lens = (ql, self.q_lens) if k_lens is None else _lengths(k_lens, "k_lens")
        if len(self.q_lens) != len(self.k_lens):
            raise RuntimeError(f"q_lens and k_lens must have the same length, got {len(self.q_lens)} and {len(self.k_lens)}")
        rl, self.rows = (None, list(range(len(self.q_lens)))) if rows is None else _lengths(rows, "rows")
        if len(self.rows) != len(self.q_lens):
            raise RuntimeError(f"rows must name one cache row per sequence, got {len(self.rows)} for {len(self.q_lens)}")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError(f"palu_b200 runs on CUDA tensors only (no CPU path); got a plan for {self.device}")
        self.info = _lib.PrefillPlanInfo()
        lib, n = _lib.load(), len(self.q_lens)
        if torch.cuda.is_available():
            if self.device.index is None:
                self.device = torch.device("cuda", torch.cuda.current_device())
            ctas = torch.cuda.get_device_properties(self.device).multi_processor_count
        else:
            ctas = 0
        size = 1 << 16
        while True:
            host = torch.empty(size, dtype=torch.uint8)
            st = lib.palu_plan_prefill(ql, kl, rl, n, int(n_q_heads), int(n_kv_heads), ctas, host.data_ptr(), size,
                                       ctypes.byref(self.info))
            if st != _lib.PALU_ERR_WORKSPACE:
                break
            size = int(self.info.bytes)
        _lib.check(st)
        self.q_tokens, self.k_tokens = int(self.info.q_tokens), int(self.info.k_tokens)
        self.n_q_heads, self.n_kv_heads = int(n_q_heads), int(n_kv_heads)
        self.max_k_len, self.max_row = int(self.info.max_k_len), int(self.info.max_row)
        self._ws_bytes, self._index = {}, None
        self.host = host[:int(self.info.bytes)]
        self.data = self.host.to(self.device)
        self._made_on = torch.cuda.current_stream(self.device)
        self._made_on.synchronize()
        self._stream = self._made_on.cuda_stream
        self.info_ptr, self.data_ptr = ctypes.byref(self.info), self.data.data_ptr()

    def workspace_bytes(self, d_v: int) -> int:
        n = self._ws_bytes.get(d_v)
        if n is None:
            n = self._ws_bytes[d_v] = int(_lib.load().palu_prefill_workspace_bytes(self.info_ptr, d_v))
        return n

    def use_on(self, stream: int) -> None:
        """Keep the plan's memory until work queued on ``stream`` is done, if that is not the stream it was made on."""
        if stream != self._stream and not torch.cuda.is_current_stream_capturing():
            for t in (self.data, self._index):
                if t is not None:
                    t.record_stream(torch.cuda.current_stream(self.device))

    def token_index(self):
        """Per packed query token its cache row and its position ([q_tokens] int64 each, on the device; laid out once): the
        queries of a sequence stand at the last of its keys' positions."""
        if self._index is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("call the plan's token_index (or run the step once) before capturing a CUDA graph with it")
            ql, kl = torch.tensor(self.q_lens), torch.tensor(self.k_lens)
            start = torch.repeat_interleave(kl - ql - (ql.cumsum(0) - ql), ql)
            host = torch.stack([torch.repeat_interleave(torch.tensor(self.rows), ql), torch.arange(self.q_tokens) + start])
            with torch.cuda.stream(self._made_on):  # as the plan's own memory: use_on knows its stream
                self._index = host.to(self.device)
            self._made_on.synchronize()
        return self._index[0], self._index[1]

    def status(self) -> int:
        """Read and clear the plan's status word: nonzero when a bounded device wait of a call expired (the rows that it
        kept from being computed are NaN)."""
        return _lib.read_status(self.data)


def _heads(t: torch.Tensor, what: str, tokens: int, heads: int, width: Optional[int], device) -> torch.Tensor:
    """A bf16 [tokens, heads, width] tensor on the plan's device, its last dimension contiguous and its rows 16-byte
    aligned (copied where they are not)."""
    shape = t.shape
    if len(shape) != 3 or shape[0] != tokens or shape[1] != heads or (width is not None and shape[2] != width):
        raise RuntimeError(f"{what} must be [{tokens}, {heads}, {width if width is not None else 'd_v'}], got {tuple(shape)}")
    if t.dtype != torch.bfloat16:
        raise RuntimeError(f"{what} must be bf16, got {t.dtype}")
    if t.device != device:
        raise RuntimeError(f"{what} is on {t.device}, the plan on {device}")
    s0, s1, s2 = t.stride()
    if s2 != 1 or s1 % 8 or s0 % 8 or s0 <= 0 or s1 <= 0 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def prefill_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: PrefillPlan, *, scale: Optional[float] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of a packed batch (palu_prefill_attn): q [q_tokens, n_q, 128], k [k_tokens, n_kv, 128] (both already
    rotated), v [k_tokens, n_kv, d_v] bf16, d_v a multiple of 16 up to 128 -> [q_tokens, n_q, d_v] bf16.

    Query i of a sequence sees its keys 0 .. i + k_len - q_len; one that sees none gives 0. What lies behind a query's
    last key does not reach its result, whatever it holds. q, k and v may be strided (slices of a fused projection);
    the products accumulate in fp32, the probabilities are rounded to bf16 for the second one."""
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        _lib.require_cuda(q, k, v, out)
    dev = plan.device
    q = _heads(q, "q", plan.q_tokens, plan.n_q_heads, HEAD_DIM, dev)
    k = _heads(k, "k", plan.k_tokens, plan.n_kv_heads, HEAD_DIM, dev)
    v = _heads(v, "v", plan.k_tokens, plan.n_kv_heads, None, dev)
    d_v = v.shape[2]
    if out is None:
        out = torch.empty(plan.q_tokens, plan.n_q_heads, d_v, dtype=torch.bfloat16, device=dev)
    elif (tuple(out.shape) != (plan.q_tokens, plan.n_q_heads, d_v) or out.dtype != torch.bfloat16 or not out.is_contiguous()
          or out.device != dev):
        raise RuntimeError(f"out must be a contiguous bf16 {(plan.q_tokens, plan.n_q_heads, d_v)} tensor on {dev}")
    else:
        at, end = out.data_ptr(), out.data_ptr() + out.nbytes
        for t in (q, k, v):
            (n, h, w), (s0, s1, _) = t.shape, t.stride()
            if n and at < t.data_ptr() + 2 * ((n - 1) * s0 + (h - 1) * s1 + w) and t.data_ptr() < end:
                raise RuntimeError("out must not overlap q, k or v")
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return prefill_attn(q, k, v, plan, scale=scale, out=out)
    need = plan.workspace_bytes(d_v)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    stream = _lib.stream_handle(dev)
    plan.use_on(stream)
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    _lib.check(_lib.load().palu_prefill_attn(
        q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], out.data_ptr(), d_v, plan.info_ptr,
        plan.data_ptr, None if ws is None else ws.data_ptr(), need, _SCALE if scale is None else float(scale), stream))
    return out


def _refuse_rebuild(dev, k_latent, v_latent, u_k, u_v, cos, sin, page_table) -> None:
    """Which of rebuild_kv's tensors is of the wrong type or on the wrong device."""
    for t, what, dtype in ((k_latent, "k_latent", torch.bfloat16), (v_latent, "v_latent", torch.bfloat16),
                           (u_k, "u_k", torch.bfloat16), (u_v, "u_v", torch.bfloat16), (cos, "cos", torch.float32),
                           (sin, "sin", torch.float32), (page_table, "page_table", None)):
        if t is not None and t.device != dev:
            _lib.require_cuda(t)
            raise RuntimeError(f"{what} is on {t.device}, the plan on {dev}")
        if t is not None and dtype is not None and t.dtype != dtype:
            raise RuntimeError(f"{what} must be {'fp32' if dtype == torch.float32 else 'bf16'}, got {t.dtype}")


def rebuild_kv(k_latent: torch.Tensor, v_latent: torch.Tensor, u_k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
               plan: PrefillPlan, *, u_v: Optional[torch.Tensor] = None, page_table: Optional[torch.Tensor] = None):
    """The packed keys and values of the plan's ``k_lens`` cached positions per sequence (palu_rebuild_kv), which
    ``prefill_attn`` takes: K = R_pos(latent U_k) [k_tokens, n_kv, 128] and V = latent U_v [k_tokens, n_kv, 128], or the V
    latents themselves [k_tokens, n_groups, r_v] without ``u_v`` (absorbed V).

    k_latent / v_latent: bf16 caches [B, n_groups, S, r], or paged [n_blocks, n_groups, block_size, r] with ``page_table``
    [rows, blocks per row] int32 (an entry outside the cache reads as zero latents); u_k [n_kv, r_k, 128], u_v [n_kv, r_v,
    128] bf16; cos / sin [>= longest k_len, 128] fp32 as the layer's tables. Sequence s reads cache row ``plan.rows[s]``.
    fp32 accumulation and rotation, one rounding to bf16."""
    dev, n_kv = plan.device, plan.n_kv_heads
    bf16, f32 = torch.bfloat16, torch.float32
    if not (k_latent.dtype == bf16 and v_latent.dtype == bf16 and u_k.dtype == bf16 and (u_v is None or u_v.dtype == bf16)
            and cos.dtype == f32 and sin.dtype == f32 and k_latent.device == dev and v_latent.device == dev
            and u_k.device == dev and (u_v is None or u_v.device == dev) and cos.device == dev and sin.device == dev
            and (page_table is None or page_table.device == dev)):
        _refuse_rebuild(dev, k_latent, v_latent, u_k, u_v, cos, sin, page_table)
    ks, vs, us = k_latent.shape, v_latent.shape, u_k.shape
    if len(ks) != 4 or len(vs) != 4 or ks[:3] != vs[:3]:
        raise RuntimeError(f"k_latent and v_latent must be [B, n_groups, S, r] with the same leading dims, got {tuple(ks)} and "
                           f"{tuple(vs)}")
    rows, n_groups, S, r_k = ks
    r_v = vs[3]
    if len(us) != 3 or us[0] != n_kv or us[1] != r_k or us[2] != HEAD_DIM:
        raise RuntimeError(f"u_k must be [{n_kv}, {r_k}, 128], got {tuple(us)}")
    if u_v is not None and tuple(u_v.shape) != (n_kv, r_v, HEAD_DIM):
        raise RuntimeError(f"u_v must be [{n_kv}, {r_v}, 128], got {tuple(u_v.shape)}")
    longest, last_row = plan.max_k_len, plan.max_row
    for t in (cos, sin):
        if t.dim() != 2 or t.shape[1] != HEAD_DIM or t.shape[0] < longest or not t.is_contiguous():
            raise RuntimeError(f"cos and sin must be contiguous fp32 [>= {longest}, 128] tables, got {tuple(t.shape)}")
    pg = None
    if page_table is not None:
        if page_table.dtype != torch.int32 or page_table.stride(-1) != 1:
            page_table = page_table.to(torch.int32).contiguous()
        pg = _lib.pages(page_table, S, rows)
        rows, S = page_table.shape[0], page_table.shape[1] * S
    if longest > S or last_row >= rows:
        raise RuntimeError(f"the plan's longest sequence ({longest}) and last cache row ({last_row}) must fit the {rows} rows of "
                           f"{S} positions")
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return rebuild_kv(k_latent, v_latent, u_k, cos, sin, plan, u_v=u_v, page_table=page_table)
    k_latent, v_latent, u_k = k_latent.contiguous(), v_latent.contiguous(), u_k.contiguous()
    k = torch.empty(plan.k_tokens, n_kv, HEAD_DIM, dtype=torch.bfloat16, device=dev)
    if u_v is not None:
        u_v = u_v.contiguous()
        v = torch.empty_like(k)
    else:
        v = torch.empty(plan.k_tokens, n_groups, r_v, dtype=torch.bfloat16, device=dev)
    stream = _lib.stream_handle(dev)
    plan.use_on(stream)
    _lib.check(_lib.load().palu_rebuild_kv(
        k_latent.data_ptr(), v_latent.data_ptr(), u_k.data_ptr(), None if u_v is None else u_v.data_ptr(), cos.data_ptr(),
        sin.data_ptr(), None if pg is None else ctypes.byref(pg), plan.info_ptr, plan.data_ptr, k.data_ptr(), v.data_ptr(), n_groups,
        r_k, r_v, S, stream))
    return k, v
