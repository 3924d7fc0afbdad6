"""GQA attention with qk-RMSNorm + RoPE fused into the QKV epilogue and a
contiguous per-sequence KV cache, on libqmoe kernels.

Mirrors ``NeuronQwen3MoEAttention`` (qwen_with_nki.py:10081-10109): QKV
projection -> per-head RMSNorm over head_dim (q_layernorm / k_layernorm,
10102-10103) -> RoPE with base ``rope_theta`` (10083-10087) -> causal GQA
attention over the KV cache ``[B, Hkv, S, D]`` (9943-9946) -> o_proj.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib, ops


def rope_tables(head_dim: int, max_pos: int, theta: float, device) -> tuple:
    """fp32 ``cos``/``sin`` ``[max_pos, head_dim/2]`` with inverse frequencies
    ``theta^(-2i/D)`` (the first half of the duplicated-half layout)."""
    inv_freq = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.int64, device=device).float() / head_dim))
    freqs = torch.arange(max_pos, device=device, dtype=torch.float32).unsqueeze(1) * inv_freq
    return freqs.cos().contiguous(), freqs.sin().contiguous()


# Decode batches of up to this many rows project with the plain GEMM into
# fp32 and finish q/k/v inside the attention launch.
FUSED_DECODE_MAX_ROWS = 64

# Chunks of up to this many query rows at a device-held start run as
# single-query decode problems (qmoe_attn_decode_chunk).
CHUNK_DECODE_MAX = 16


@dataclass
class SharedPrefix:
    """Keys and values of the tokens that every sequence of a batch starts with,
    held once: ``k``, ``v`` bf16 ``[Hkv, P_max, D]``, of which ``length`` entries."""

    k: torch.Tensor
    v: torch.Tensor
    length: int


class KVCache:
    """Contiguous K/V cache of one layer: ``[B, Hkv, S_max, D]`` bf16 each.

    Unpacks like the reference's ``(K, V)`` present-key-value tuple
    (``k, v = cache``), and :meth:`wrap` takes such a tuple back without a copy.

    With a ``prefix`` the rows hold only what follows it: a token's cache index
    (and the ``positions`` of :meth:`Attention.forward`) counts from the
    prefix's end, and the caller's RoPE tables start there too."""

    prefix: Optional[SharedPrefix] = None

    def __init__(self, B: int, n_kv: int, S_max: int, head_dim: int, device):
        self.k = torch.zeros(B, n_kv, S_max, head_dim, dtype=torch.bfloat16, device=device)
        self.v = torch.zeros_like(self.k)

    @classmethod
    def wrap(cls, kv) -> "KVCache":
        """A :class:`KVCache` as is, or a ``(K, V)`` pair of contiguous bf16
        ``[B, Hkv, S_max, D]`` device tensors viewed as one (no copy)."""
        if isinstance(kv, KVCache):
            return kv
        if not isinstance(kv, (tuple, list)) or len(kv) != 2:
            raise ValueError("past_key_value must be a KVCache or a (K, V) pair")
        k, v = kv
        for name, t in (("K", k), ("V", v)):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.bfloat16 or t.dim() != 4 \
                    or not t.is_contiguous() or t.device.type != "cuda":
                raise ValueError(f"past_key_value {name} must be a contiguous bf16 [B, Hkv, S_max, D] GPU tensor")
        if k.shape != v.shape:
            raise ValueError("past_key_value K and V shapes differ")
        c = cls.__new__(cls)
        c.k, c.v = k, v
        return c

    @property
    def capacity(self) -> int:
        return self.k.shape[2]

    def __iter__(self):
        return iter((self.k, self.v))

    def __len__(self) -> int:
        return 2

    def __getitem__(self, i):
        return (self.k, self.v)[i]


def check_budget(budget: int, recent: int, sink: int, slack: int = 1) -> None:
    if budget <= 0 or recent < 0 or sink < 0 or recent + sink > budget or slack < 1:
        raise ValueError(f"need 0 <= recent + sink <= budget and at least one slot past it (budget={budget}, "
                         f"recent={recent}, sink={sink}, slack={slack})")


def default_recent(budget: int, sink: int) -> int:
    """A quarter of the budget, and no more than the sinks leave of it."""
    return max(0, min(budget // 4, budget - sink))


class CacheBudget:
    """What the bounded caches of all layers have in common: how many entries a
    row keeps (``budget``: the first ``sink`` positions, the ``recent`` last
    ones and those with the most attention weight), the slots past it that
    decode steps fill before the next eviction, and where each row stands.

    ``slots[b]`` (device) is the slot of row b's next token and ``ctx`` is
    ``slots + 1``, the entries its step sees; ``used`` is the same on the host,
    so no step has to ask the device.  ``lengths`` are a prompt's real tokens."""

    def __init__(self, B: int, budget: int, recent: int, sink: int, slack: int, device):
        check_budget(budget, recent, sink, slack)
        self.budget, self.recent, self.sink, self.capacity = budget, recent, sink, budget + slack
        self.slots = torch.zeros(B, dtype=torch.int32, device=device)
        self.ctx = torch.ones(B, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(B, dtype=torch.int32, device=device)
        self.used = [0] * B
        self._prompt = None

    def prompt_cache(self, n_kv: int, S: int, head_dim: int):
        """Scratch cache of a whole prompt (one for all layers, which run one
        after another) with its scores at zero and its positions."""
        B, dev = len(self.used), self.slots.device
        p = self._prompt
        if p is None or p[0].k.shape[1] != n_kv or p[0].capacity < S:
            c = KVCache(B, n_kv, S, head_dim, dev)
            pos = torch.arange(S, dtype=torch.int32, device=dev).repeat(B, n_kv, 1)
            p = self._prompt = (c, torch.empty(B, n_kv, S, device=dev), pos)
        p[1].zero_()
        return p

    def begin(self, lengths: list) -> None:
        """A prompt of ``lengths[b]`` real tokens a row comes next."""
        self.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        self._stand([min(int(n), self.budget) for n in lengths])

    def _stand(self, used: list) -> None:
        self.used = used
        self.slots.copy_(torch.tensor(used, dtype=torch.int32))
        self.ctx.copy_(self.slots + 1)

    def advance(self) -> None:
        """After a step, on the host (the step itself moves ``slots`` and ``ctx``)."""
        self.used = [n + 1 for n in self.used]

    def make_room(self, caches) -> None:
        """Before a step: evicts in every layer once a row's slots are full."""
        if max(self.used) < self.capacity:
            return
        for c in caches:
            ops.kv_evict(c.k, c.v, c.scores, c.slot_pos, self.slots, self.budget, self.recent, self.sink)
        self._stand([min(n, self.budget) for n in self.used])


class BoundedKVCache(KVCache):
    """One layer's cache of at most ``state.budget`` entries per row and kv head
    between evictions, whose slots are not positions: ``scores`` (f32) and
    ``slot_pos`` (i32) ``[B, Hkv, capacity]`` hold each entry's accumulated
    attention weight and position."""

    def __init__(self, state: CacheBudget, n_kv: int, head_dim: int):
        B, dev = len(state.used), state.slots.device
        super().__init__(B, n_kv, state.capacity, head_dim, dev)
        self.state = state
        self.scores = torch.zeros(B, n_kv, state.capacity, device=dev)
        self.slot_pos = torch.full((B, n_kv, state.capacity), -1, dtype=torch.int32, device=dev)


class Attention:
    """One layer's attention.  ``forward`` adds ``o_proj(attn(x))`` to the fp32
    residual stream in place (the residual add of qwen_with_nki.py:10200 fused
    into the o_proj epilogue)."""

    def __init__(self, wqkv, q_norm, k_norm, wo, n_q: int, n_kv: int, head_dim: int, eps: float):
        self.wqkv, self.q_norm, self.k_norm, self.wo = wqkv, q_norm, k_norm, wo
        self.n_q, self.n_kv, self.head_dim, self.eps = n_q, n_kv, head_dim, eps
        self.scale = 1.0 / math.sqrt(head_dim)
        self._ws = {}

    def _decode_ws(self, B: int, cache: KVCache, device) -> torch.Tensor:
        ws = self._ws.get((B, cache.capacity))
        if ws is None:
            ws = ops.attn_decode_workspace(B, self.n_q, self.head_dim, cache.capacity, device)
            self._ws[(B, cache.capacity)] = ws
        return ws

    def _skinny_decode(self, x: torch.Tensor, B: int) -> bool:
        """Whether a decode step past the GEMV's rows projects with ``ops.gemm``.
        Above 16 rows some of its kernels copy both operands by LDS-DMA (16
        bytes a lane, 32-bit offsets); ``qkv_norm_rope`` takes operands that are
        off that alignment, or too large, through registers."""
        return (0 < B <= FUSED_DECODE_MAX_ROWS and x.shape[1] in ops.SKINNY_K
                and x.data_ptr() % 16 == 0 and self.wqkv.data_ptr() % 16 == 0
                and self.wqkv.numel() * self.wqkv.element_size() < 2**31)

    def forward(self, x: torch.Tensor, residual: torch.Tensor, positions: torch.Tensor, B: int, S: int,
                cache: KVCache, rope_cos: torch.Tensor, rope_sin: torch.Tensor, start=0,
                max_ctx: Optional[int] = None, norm: Optional[tuple] = None,
                post_norm: Optional[tuple] = None) -> torch.Tensor:
        """``x[B*S, H]`` bf16 (input-normed), ``residual[B*S, H]`` f32 (updated
        in place), ``positions[B*S]`` i32 (RoPE position == cache index).

        S > 1: causal prefill of a chunk starting at cache index ``start`` (an
        int, or an int32 ``[1]`` device tensor for graph replays at any position).
        S == 1: decode; row b sees cache entries ``[0, positions[b]]`` (at most
        the first ``max_ctx`` when a context bucket is given), on every path.
        Up to ``FUSED_DECODE_MAX_ROWS`` decode rows the finish runs inside the
        attention launch (``attn_decode_fused``), past the GEMV's rows only
        with 16-byte aligned ``x`` and ``wqkv``.
        ``norm = (rms_w, eps)``: ``x`` is the fp32 residual row itself (B*S == 1)
        and the input RMSNorm is fused into the QKV GEMV.
        ``post_norm = (rms_w, eps)``: returns ``bf16(rmsnorm(residual) * rms_w)``
        of the updated residual, computed with the o_proj's residual add
        (instead of the residual itself).

        A cache with a ``prefix``: positions count from the prefix's end, every
        query also sees the prefix (``attn_shared``).  A
        :class:`BoundedKVCache`: a decode row's entry goes to slot
        ``state.slots[b]`` and the weights of its attention to the scores; a
        prompt (``start`` 0, ``state.lengths`` real tokens a row) is attended
        in full and then cut down to the budget.
        """
        if cache.prefix is not None or isinstance(cache, BoundedKVCache):
            o = self._special(x, positions, B, S, cache, rope_cos, rope_sin, start, max_ctx, norm)
        else:
            o = self._plain(x, positions, B, S, cache, rope_cos, rope_sin, start, max_ctx, norm)
        key = ("oproj", o.shape[0])
        if key not in self._ws:  # split-K scratch for prefill-size token counts (None: not split)
            self._ws[key] = ops.gemm_workspace(o.shape[0], self.wo.shape[0], self.wo.shape[1], x.device)
        if post_norm is not None:
            return ops.gemm_add_rmsnorm(o, self.wo, residual, post_norm[0], post_norm[1], workspace=self._ws[key])
        ops.gemm(o, self.wo, _lib.GEMM_ADD_F32, out=residual, workspace=self._ws[key])
        return residual

    def _plain(self, x, positions, B, S, cache, rope_cos, rope_sin, start, max_ctx, norm) -> torch.Tensor:
        """Attention outputs ``[B*S, Hq*D]`` over a contiguous cache."""
        n_ws = ops.qkv_norm_rope_workspace(B * S, x.shape[1], self.n_q, self.n_kv, self.head_dim)
        n_raw = n_ws
        if S == 1 and n_ws == 0 and self._skinny_decode(x, B):
            n_raw = B * self.wqkv.shape[0] * 4
        qws = self._ws.get(("qkv", B * S))
        if qws is None or qws.numel() * 4 < n_raw:
            qws = torch.empty(max(n_raw // 4, 1), dtype=torch.float32, device=x.device)
            self._ws[("qkv", B * S)] = qws
        if norm is not None and (B * S != 1 or n_ws == 0):
            raise ValueError("the fused input norm takes one fp32 row on the GEMV path")
        if S == 1 and n_raw > 0:
            # decode: raw projection, then finish + attention in one launch
            raw = qws[: n_raw // 4].view(B, -1)
            if norm is not None:
                ops.gemv_rmsnorm(x, norm[0], norm[1], self.wqkv, _lib.GEMM_STORE_F32, out=raw)
            else:
                ops.gemm(x, self.wqkv, _lib.GEMM_STORE_F32, out=raw)
            o = ops.attn_decode_fused(raw, self.q_norm, self.k_norm, rope_cos, rope_sin, positions, self.n_q,
                                      self.n_kv, cache.k, cache.v, self.eps, self.scale,
                                      self._decode_ws(B, cache, x.device), max_ctx=max_ctx)
        else:
            q = ops.qkv_norm_rope(x, self.wqkv, self.q_norm, self.k_norm, rope_cos, rope_sin, positions, B, S,
                                  self.n_q, self.n_kv, cache.k, cache.v, self.eps, workspace=qws)
            if S > 1 and isinstance(start, torch.Tensor) and B * S <= CHUNK_DECODE_MAX:
                # a few-token chunk at a device-held position (speculative verification):
                # one decode problem per query spreads the K/V stream over many CUs
                ws = self._ws.get(("chunk", B * S, cache.capacity))
                if ws is None:
                    ws = ops.attn_decode_workspace(B * S, self.n_q, self.head_dim, cache.capacity, x.device)
                    self._ws[("chunk", B * S, cache.capacity)] = ws
                o = ops.attn_decode_chunk(q.view(B * S, self.n_q, self.head_dim), cache.k, cache.v, B, S, start,
                                          self.scale, ws)
            elif S > 1:
                aws = None
                if not isinstance(start, torch.Tensor):
                    aws = self._ws.get(("prefill", B, S))
                    if aws is None:
                        aws = ops.attn_prefill_workspace(B, S, self.n_q, self.head_dim, x.device)
                        self._ws[("prefill", B, S)] = aws
                o = ops.attn_prefill(q, cache.k, cache.v, B, S, start, self.scale, workspace=aws)
            else:
                o = ops.attn_decode(q.view(B, self.n_q, self.head_dim), cache.k, cache.v, positions + 1, self.scale,
                                    self._decode_ws(B, cache, x.device), max_ctx=max_ctx)
        return o

    def _special(self, x, positions, B, S, cache, rope_cos, rope_sin, start, max_ctx, norm) -> torch.Tensor:
        """Attention outputs ``[B*S, Hq*D]`` over a shared prefix or a bounded cache."""
        bounded = isinstance(cache, BoundedKVCache)
        if isinstance(start, torch.Tensor):
            raise ValueError("a chunk at a device-held position needs a contiguous cache without a prefix")
        if S > 1:
            if norm is not None:
                raise ValueError("the fused input norm takes one fp32 row on the GEMV path")
            if bounded and start != 0:
                raise ValueError("a bounded cache takes a prompt from its first token on")
            # past it qkv_norm_rope writes neither queries nor entries
            limit = rope_cos.shape[0] if bounded else min(rope_cos.shape[0], cache.capacity)
            if start < 0 or start + S > limit:
                raise ValueError(f"need 0 <= start and start + S <= {limit} (start={start}, S={S})")
            n = ops.qkv_norm_rope_workspace(B * S, x.shape[1], self.n_q, self.n_kv, self.head_dim)
            ws = torch.empty(n // 4, dtype=torch.float32, device=x.device) if n > 0 else None
            own, scores, pos = cache.state.prompt_cache(self.n_kv, S, self.head_dim) if bounded else (cache, None, None)
            q = ops.qkv_norm_rope(x, self.wqkv, self.q_norm, self.k_norm, rope_cos, rope_sin, positions, B, S,
                                  self.n_q, self.n_kv, own.k, own.v, self.eps, workspace=ws)
            if not bounded:
                ctx = positions.view(B, S)[:, 0] + 1
                return ops.attn_shared(q, cache.prefix.k, cache.prefix.v, cache.k, cache.v, ctx, B, S,
                                       cache.prefix.length, self.scale, max_ctx=min(cache.capacity, start + S))
            st = cache.state
            o = ops.attn_prefill_scored(q, own.k, own.v, scores, B, S, 0, st.lengths, self.scale)
            ops.kv_evict(own.k, own.v, scores, pos, st.lengths, st.budget, st.recent, st.sink,
                         out=(cache.k, cache.v, cache.scores, cache.slot_pos))
            return o
        gemv = ops.qkv_norm_rope_workspace(B, x.shape[1], self.n_q, self.n_kv, self.head_dim) > 0
        if norm is not None:
            raw = ops.gemv_rmsnorm(x, norm[0], norm[1], self.wqkv, _lib.GEMM_STORE_F32)
        elif gemv or self._skinny_decode(x, B):
            raw = ops.gemm(x, self.wqkv, _lib.GEMM_STORE_F32)
        else:
            raw = self._raw_of_any(x) if bounded else None
        if not bounded:
            if raw is None:
                q = ops.qkv_norm_rope(x, self.wqkv, self.q_norm, self.k_norm, rope_cos, rope_sin, positions, B, 1,
                                      self.n_q, self.n_kv, cache.k, cache.v, self.eps)
            else:
                q = ops.kv_append(raw, self.q_norm, self.k_norm, rope_cos, rope_sin, positions, positions, self.n_q,
                                  self.n_kv, cache.k, cache.v, self.eps)
            return ops.attn_shared(q, cache.prefix.k, cache.prefix.v, cache.k, cache.v, positions + 1, B, 1,
                                   cache.prefix.length, self.scale, max_ctx=max_ctx)
        st = cache.state
        q = ops.kv_append(raw, self.q_norm, self.k_norm, rope_cos, rope_sin, positions, st.slots, self.n_q, self.n_kv,
                          cache.k, cache.v, self.eps, scores=cache.scores, slot_pos=cache.slot_pos)
        return ops.attn_decode_scored(q, cache.k, cache.v, st.ctx, cache.scores, self.scale, max_ctx=max_ctx)

    def _raw_of_any(self, x: torch.Tensor) -> torch.Tensor:
        """The raw projection of rows that ``_skinny_decode`` leaves to
        ``qkv_norm_rope``, whose cache row is the position and so no slot of a
        bounded cache.  ``ops.gemm`` takes them with operands on its alignment
        (copies of those that are not), ``wqkv`` in pieces below 2 GiB, and no
        fewer rows than its tiles have where the GEMV does not take the hidden
        size."""
        rows, H = x.shape
        if rows < 17 and H % 512:
            x = torch.nn.functional.pad(x, (0, 0, 0, 17 - rows))
        elif x.data_ptr() % 16:
            x = x.clone()
        pieces = self.wqkv.chunk(1 + self.wqkv.numel() * self.wqkv.element_size() // 2**31)
        raw = [ops.gemm(x, w.clone() if w.data_ptr() % 16 else w, _lib.GEMM_STORE_F32) for w in pieces]
        return (raw[0] if len(raw) == 1 else torch.cat(raw, 1))[:rows]
