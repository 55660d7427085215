"""``LatentAttentionLayer``: the reference's model layer (latent_attn/__init__.py:41-198 of
anishesg/latent-attn) on this library's kernels.

Same parameters (names, shapes, initialisation), same ``forward(x, kv_cache)`` contract and
result: ``q_absorbed = x @ W_Q_absorbed^T`` and ``q_rope = x @ W_Q_rope^T`` (not rotated, as in
the reference), the fused absorbed decode with W_UV in the cache's dtype, then ``@ W_O^T``
(latent_attn/__init__.py:110-145). The three projections run on the tcgen05 projection GEMM
(``_C.linear``) with weights and activations in the cache's 16-bit type; the decode runs through
``mla_decode``.

``decode_step`` is the batched form for a serving loop: B tokens (B <= 256), each attending to
its own sequence (variable lengths, contiguous or paged cache), optionally with the query's RoPE
part rotated to the token's position.

``prefix_decode_step`` is a serving step over a ``SharedPrefixBatch``: requests in groups that share a
prefix, a cache of normalised rows with rotated keys, and optionally each request's own low-rank
adapters on the projections.

``reference_forward`` is the reference's pure-torch check with its shape error corrected: the
reference multiplies ``(H, d_c) @ (H * dn, d_c)`` (latent_attn/__init__.py:183), which cannot
run. Since ``q_absorbed`` already lives in the latent space, the nope score is
``q_absorbed . c_t`` (the absorbed identity the fused path computes), and the rope score and
softmax are the reference's.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn

from . import MLAConfig, _C
from .synthetic import build_rope_tables


def _rotate_half(q: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    half = q.shape[-1] // 2
    q0, q1 = q[..., :half], q[..., half:]
    return torch.cat([q0 * cos - q1 * sin, q0 * sin + q1 * cos], dim=-1)


class SharedPrefixBatch:
    """Index tensors of a batch of B requests in groups, each group's requests after one prefix.

    ``group_sizes``: requests per group (they sum to B; the batch is in group order).
    ``prefix_lens``: rows of each group's prefix; ``own_lens``: rows that each request has after it so
    far; ``max_own_len``: the most it may come to have. The rows lie in the cache either from
    ``prefix_offsets`` (groups) and ``own_offsets`` (B) on, or in pages of ``page_rows`` rows (a multiple
    of 64, of which every prefix length is a multiple) listed by ``prefix_table`` and ``own_table``.
    All are host sequences (tables: lists of lists); the tensors are built once, for as long as the
    batch keeps its requests.

    The lengths advance on the device, in place, so a captured step advances with every replay. A step on
    a batch with a full request is refused on the host, which counts the steps that it runs itself;
    a replay drops the token of a full request (its lengths and rows stay, its output means nothing) and
    sets bit 0 of ``status`` (int32, on the device)."""

    def __init__(self, cfg: MLAConfig, device, group_sizes, prefix_lens, own_lens, max_own_len: int, *,
                 prefix_offsets=None, own_offsets=None, prefix_table=None, own_table=None, page_rows: int = 0) -> None:
        B, groups = sum(group_sizes), len(group_sizes)
        if len(prefix_lens) != groups or len(own_lens) != B:
            raise RuntimeError("prefix_lens needs one entry per group and own_lens one per request")
        if max(own_lens, default=0) > max_own_len:
            raise RuntimeError("own_lens exceed max_own_len")
        paged = page_rows > 0
        if paged != (own_table is not None) or paged != (prefix_table is not None) or paged == (own_offsets is not None) \
                or paged == (prefix_offsets is not None):
            raise RuntimeError("give prefix_offsets and own_offsets, or page_rows with prefix_table and own_table")

        def ints(v, dtype=torch.int32):
            return torch.tensor(v, dtype=dtype, device=device)

        self.batch, self.page_rows = B, page_rows
        self.max_prefix_len, self.max_own_len = max(prefix_lens, default=0), max_own_len
        self.max_positions = self.max_prefix_len + max_own_len
        first = [n for n, size in zip(prefix_lens, group_sizes) for _ in range(size)]   # a request's first own position
        starts = [0]
        for size in group_sizes:
            starts.append(starts[-1] + size)
        self.group_starts, self.prefix_lens, self.first = ints(starts), ints(prefix_lens), ints(first)
        self.own_lens = ints(own_lens)
        # where each request's next token goes; max_positions, where the append drops it, once it is full
        self.positions = ints([f + n if n < max_own_len else self.max_positions for f, n in zip(first, own_lens)])
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self._next = torch.empty_like(self.positions)
        self._limits = ints([f + max_own_len for f in first])
        self._full = torch.full_like(self.positions, self.max_positions)
        self._room = max_own_len - max(own_lens, default=0)   # steps until the longest request is full
        self.cu_tokens = ints(range(B + 1))
        self.prefix_offsets = self.own_offsets = self.row_offsets = None
        self.prefix_table = self.own_table = self.row_table = None
        if paged:
            if any(n % page_rows for n in prefix_lens):
                raise RuntimeError("prefix lengths must be multiples of page_rows")
            self.prefix_table, self.own_table = ints(prefix_table), ints(own_table)
            pages = self.max_prefix_len // page_rows + self.own_table.size(1)
            rows = [[0] * (f // page_rows) + list(own) for f, own in zip(first, own_table)]
            self.row_table = ints([r + [0] * (pages - len(r)) for r in rows])   # page of each position
        else:
            self.prefix_offsets, self.own_offsets = ints(prefix_offsets, torch.int64), ints(own_offsets, torch.int64)
            self.row_offsets = self.own_offsets - self.first                    # row of position 0
        # the one record of a finished softmax (maximum 0, sum 1) that the value projection takes
        self.part_ml = torch.tensor([0.0, 1.0], device=device).expand(1, B, cfg.num_heads, 2).contiguous()

    def advance(self) -> None:
        """The appended tokens become part of the lengths."""
        if not (self.positions.is_cuda and torch.cuda.is_current_stream_capturing()):
            self._room -= 1
        torch.sub(self._next, self.first, out=self.own_lens).clamp_(max=self.max_own_len)
        torch.where(self._next < self._limits, self._next, self._full, out=self.positions)


class LatentAttentionLayer(nn.Module):
    """Multi-head latent attention with the absorbed query projection (drop-in for the reference's
    ``latent_attn.LatentAttentionLayer``)."""

    def __init__(self, cfg: MLAConfig, max_seq_len: int = 8192) -> None:
        super().__init__()
        self.cfg = cfg
        self.max_seq_len = max_seq_len
        H, dc, dR, dn, dv, dm = (cfg.num_heads, cfg.kv_lora_rank, cfg.qk_rope_head_dim, cfg.qk_nope_head_dim,
                                 cfg.v_head_dim, cfg.d_model)
        self.W_Q_absorbed = nn.Parameter(torch.empty(H * dc, dm))
        self.W_Q_rope = nn.Parameter(torch.empty(H * dR, dm))
        self.W_UK = nn.Parameter(torch.empty(H * dn, dc))
        self.W_UV = nn.Parameter(torch.empty(H * dv, dc))
        self.W_O = nn.Parameter(torch.empty(dm, H * dv))
        self._init_weights()
        cos, sin = build_rope_tables(max_seq_len, dR)
        self.register_buffer("rope_cos", cos)
        self.register_buffer("rope_sin", sin)
        self._lowp = {}

    def _init_weights(self) -> None:
        std = 0.02
        nn.init.normal_(self.W_Q_absorbed, std=std)
        nn.init.normal_(self.W_Q_rope, std=std)
        nn.init.normal_(self.W_UK, std=std)
        nn.init.normal_(self.W_UV, std=std)
        nn.init.normal_(self.W_O, std=std / math.sqrt(2.0))

    @staticmethod
    def from_config(cfg: MLAConfig, max_seq_len: int = 8192) -> "LatentAttentionLayer":
        return LatentAttentionLayer(cfg, max_seq_len)

    def _weight(self, name: str, dtype: torch.dtype) -> torch.Tensor:
        """16-bit copy of a parameter, refreshed when the parameter changes."""
        p = getattr(self, name)
        key = (name, dtype)
        hit = self._lowp.get(key)
        stamp = (p.data_ptr(), p._version, p.device)
        if hit is None or hit[0] != stamp:
            hit = (stamp, p.detach().to(dtype).contiguous())
            self._lowp[key] = hit
        return hit[1]

    def _w_uv_fp16(self) -> torch.Tensor:
        return self._weight("W_UV", torch.float16)

    def _w_uk_fp16(self) -> torch.Tensor:
        return self._weight("W_UK", torch.float16)

    def forward(self, x: torch.Tensor, kv_cache: torch.Tensor) -> torch.Tensor:
        """One decode token: ``x`` (d_model,) or (1, d_model), ``kv_cache`` (seq_len, d_c + d_R)
        fp16/bf16 on CUDA. Returns (d_model,) fp32."""
        if x.dim() == 2:
            x = x.squeeze(0)
        assert x.dim() == 1 and x.size(0) == self.cfg.d_model
        return self.decode_step(x.unsqueeze(0), kv_cache)[0]

    def decode_step(self, x: torch.Tensor, kv_cache: torch.Tensor, *, seq_lens: Optional[torch.Tensor] = None,
                    kv_offsets: Optional[torch.Tensor] = None, max_seq_len: Optional[int] = None,
                    seq_lens_host=None, page_table: Optional[torch.Tensor] = None, page_rows: int = 0,
                    positions: Optional[torch.Tensor] = None, rope_tables: bool = True,
                    workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """B decode tokens: ``x`` (B, d_model) -> (B, d_model) fp32.

        Token b attends to its sequence of ``kv_cache`` (``seq_lens`` / ``kv_offsets`` /
        ``page_table`` as in ``mla_decode``; without them the B sequences are ``kv_cache.size(0) //
        B`` rows each). ``positions`` (B,) int: rotate the query's RoPE part to these positions
        (the reference leaves it unrotated). ``rope_tables=False`` lets the kernels compute the
        cache's RoPE on the fly instead of reading the layer's tables."""
        from .functional import mla_decode
        cfg = self.cfg
        H, dc, dR, dv = cfg.num_heads, cfg.kv_lora_rank, cfg.qk_rope_head_dim, cfg.v_head_dim
        dt = kv_cache.dtype
        B = x.size(0)
        xh = x.to(dt).contiguous()
        q_abs = _C.linear(xh, self._weight("W_Q_absorbed", dt)).view(B, H, dc)
        q_r = _C.linear(xh, self._weight("W_Q_rope", dt)).view(B, H, dR)
        if positions is not None:
            # the table builder's angles (latent_attn/__init__.py:31-38) at each token's position
            dims = torch.arange(dR // 2, dtype=torch.float32, device=x.device)
            freqs = 1.0 / (10000.0 ** (2.0 * dims / dR))
            ang = positions.to(device=x.device, dtype=torch.float32)[:, None] * freqs[None, :]
            q_r = _rotate_half(q_r, ang.cos()[:, None, :], ang.sin()[:, None, :]).contiguous()
        if max_seq_len is None:
            max_seq_len = kv_cache.size(0) // B if seq_lens is None else int(self.max_seq_len)
        if rope_tables:
            need = max_seq_len
            if need > self.rope_cos.size(0):
                cos, sin = build_rope_tables(need, dR, device=kv_cache.device)
            else:
                cos = self.rope_cos[:need].to(kv_cache.device).contiguous()
                sin = self.rope_sin[:need].to(kv_cache.device).contiguous()
        else:
            cos = sin = None
        o = mla_decode(kv_cache, q_r, self._weight("W_UV", dt), cos, sin, cfg, q_absorbed=q_abs.contiguous(),
                       seq_lens=seq_lens, kv_offsets=kv_offsets, max_seq_len=max_seq_len,
                       seq_lens_host=seq_lens_host, page_table=page_table, page_rows=page_rows, workspace=workspace)
        return _C.linear(o.view(B, H * dv).to(dt), self._weight("W_O", dt))

    def _project(self, name: str, x: torch.Tensor, adapters, adapter_ids) -> torch.Tensor:
        """``x @ W^T`` in x's type, with the tokens' adapters where there are some for this projection."""
        W = self._weight(name, x.dtype)
        if not adapters or name not in adapters:
            return _C.linear(x, W).to(x.dtype)
        lora_a, lora_b, scales = adapters[name]
        return _C.linear_lora(x, W, lora_a, lora_b, adapter_ids, scales=scales)

    def prefix_decode_step(self, x: torch.Tensor, c: torch.Tensor, k_rope: torch.Tensor, kv_cache: torch.Tensor,
                           batch: SharedPrefixBatch, *, norm_weight: Optional[torch.Tensor] = None,
                           norm_eps: float = 1e-6, adapters=None,
                           adapter_ids: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One token of each of ``batch``'s requests: ``x`` (B, d_model) -> (B, d_model) in the cache's type.

        The tokens' latents ``c`` (B, d_c) and keys ``k_rope`` (B, d_R) are appended to the cache, normalised
        (with ``norm_weight``) and rotated to their positions, and ``batch``'s lengths advance. Each token then
        attends to its group's prefix, which is read once for the whole group, and to its request's own rows.
        The step can be captured in a CUDA graph (after one that was not: it lays the weights out).
        ``kv_cache`` (rows, d_c + d_R) holds rows as ``mla_cache_append_rope`` writes them.

        ``adapters``: per projection ("W_Q_absorbed", "W_Q_rope", "W_O") a tuple of ``lora_a``, ``lora_b`` and
        ``scales`` (or None) as ``linear_lora`` takes them; ``adapter_ids`` (B,) int32 picks each token's. Up to
        256 requests where a projection has no adapters."""
        from .functional import mla_cache_append_rope, mla_prefix_decode
        cfg = self.cfg
        H, dc, dR, dv = cfg.num_heads, cfg.kv_lora_rank, cfg.qk_rope_head_dim, cfg.v_head_dim
        dt, B = kv_cache.dtype, batch.batch
        if tuple(x.shape) != (B, cfg.d_model):
            raise RuntimeError(f"x must be ({B}, {cfg.d_model})")
        if batch._room < 1:
            raise RuntimeError("a request has max_own_len rows already")
        if adapters and adapter_ids is None:
            raise RuntimeError("adapters need adapter_ids")
        xh = x.to(dt).contiguous()
        q_abs = self._project("W_Q_absorbed", xh, adapters, adapter_ids).view(B, H, dc)
        q_r = self._project("W_Q_rope", xh, adapters, adapter_ids).view(B, H, dR)
        tables = {}
        if batch.max_positions <= self.rope_cos.size(0):
            tables = {"rope_cos": self.rope_cos, "rope_sin": self.rope_sin}
        mla_cache_append_rope(kv_cache, c.to(dt), k_rope.to(dt), batch.cu_tokens, batch.positions, batch.max_positions, cfg,
                              norm_weight=norm_weight, norm_eps=norm_eps, kv_offsets=batch.row_offsets,
                              page_table=batch.row_table, page_rows=batch.page_rows, q_rope=q_r, q_out=q_r,
                              new_lens=batch._next, status=batch.status, **tables)
        batch.advance()
        o = mla_prefix_decode(kv_cache, q_abs, q_r, cfg, group_starts=batch.group_starts, prefix_lens=batch.prefix_lens,
                              max_prefix_len=batch.max_prefix_len, seq_lens=batch.own_lens, max_seq_len=batch.max_own_len,
                              prefix_offsets=batch.prefix_offsets, kv_offsets=batch.own_offsets,
                              prefix_table=batch.prefix_table, page_table=batch.own_table, page_rows=batch.page_rows)
        o = _C.mla_combine_partials(batch.part_ml, o.float().unsqueeze(0), self._weight("W_UV", dt), cfg.d_model, dc,
                                    cfg.qk_nope_head_dim, dR, H, dv)
        return self._project("W_O", o.view(B, H * dv).to(dt), adapters, adapter_ids)

    def reference_forward(self, x: torch.Tensor, kv_cache: torch.Tensor) -> torch.Tensor:
        """Pure-torch fp32 decode of one token (the reference's check, shape error corrected)."""
        if x.dim() == 2:
            x = x.squeeze(0)
        cfg = self.cfg
        S = kv_cache.size(0)
        c_t = kv_cache[:, :cfg.kv_lora_rank].float()
        k_rope = kv_cache[:, cfg.kv_lora_rank:].float()
        cos = self.rope_cos[:S].float().to(kv_cache.device)
        sin = self.rope_sin[:S].float().to(kv_cache.device)
        K_rope = _rotate_half(k_rope, cos, sin)
        xf = x.float()
        q_abs = (xf @ self.W_Q_absorbed.float().T).view(cfg.num_heads, cfg.kv_lora_rank)
        q_r = (xf @ self.W_Q_rope.float().T).view(cfg.num_heads, cfg.qk_rope_head_dim)
        scale = 1.0 / math.sqrt(cfg.qk_nope_head_dim + cfg.qk_rope_head_dim)
        scores = (q_abs @ c_t.T + q_r @ K_rope.T) * scale
        attn = torch.softmax(scores, dim=-1)
        o_lat = attn @ c_t                                                        # (H, d_c)
        W_UV = self.W_UV.float().view(cfg.num_heads, cfg.v_head_dim, cfg.kv_lora_rank)
        out = torch.einsum("hc,hjc->hj", o_lat, W_UV)                             # (H, dv)
        return out.reshape(-1) @ self.W_O.float().T
