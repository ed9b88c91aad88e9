"""The parts of a pre-norm decoder layer in 8 bits: rows of the stream normed into 8-bit integers with a scale each, projections
as products of such rows with 8-bit weights (a scale per output channel), keys and values cached as 8-bit integers with a scale
per page and head. The weights are made from the checkpoint's as they are loaded, one after the other; everything between the products (norm,
rotation, softmax, activation, the residual stream) is in the model dtype or 32-bit as in the plain parts.

``eight_bit(spec)`` puts these parts in the place of a model's plain ones. Upstream has no counterpart.
"""

from __future__ import annotations

from dataclasses import dataclass, replace
from typing import Any, Mapping

import torch

from ..config.base import ModelSpec, PartSpec, UnsupportedConfigError
from ..kernels import ops
from .attention import GQAAttention
from .base import EVERY_STEP, PagedNeed, ResidualStream, StepContext, TensorSpec, register_feed_forward, register_mixer, register_norm
from .mlp import SwiGLU
from .norm import RMSNorm


@dataclass
class Int8Rows:
    """Rows as codes ``[T, int8_width(size)]`` and scales ``[T]``."""

    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def num_rows(self) -> int:
        return self.codes.shape[0]


def _take_rows(t: int, size: int, ctx: StepContext) -> Int8Rows:
    return Int8Rows(ctx.arena.take((t, ops.int8_width(size)), torch.int8), ctx.arena.take((t,), torch.float32))


class Int8Weight:
    """A projection's matrix ``[N, K]`` as codes and a scale per row."""

    def __init__(self, w: torch.Tensor) -> None:
        self.codes, self.scales = ops.int8_weight(w)

    @classmethod
    def of(cls, w: "torch.Tensor | Int8Weight") -> "Int8Weight":
        """A weight as it was loaded: as codes already, or as the matrix they are made from."""
        return w if isinstance(w, cls) else cls(w)

    def project(self, x: Int8Rows, ctx: StepContext, rows: int | None = None) -> torch.Tensor:
        """``x w^T`` in the model dtype; ``rows``: of the first so many rows of ``w`` only."""
        codes, scales = (self.codes, self.scales) if rows is None else (self.codes[:rows], self.scales[:rows])
        out = ctx.arena.take((x.num_rows, codes.shape[0]), ctx.dtype)
        ops.gemm_int8(x.codes, x.scales, codes, scales, out)
        return out


def _projections_in_8_bits(specs: list[TensorSpec]) -> list[TensorSpec]:
    return [replace(s, becomes=Int8Weight) if len(s.shape) == 2 else s for s in specs]


class Int8RMSNorm(RMSNorm):
    """An ``RMSNorm`` in front of 8-bit projections: 32-bit throughout, rounded once, to the codes."""

    recordable = EVERY_STEP
    folds_stream_input = False

    def forward(self, stream: ResidualStream, ctx: StepContext) -> Int8Rows:
        if stream.post is not None or stream.second is not None or stream.extra is not None or self.unit_offset:
            raise NotImplementedError("an 8-bit norm adds one plain pending output to the stream")
        out = _take_rows(stream.resid.shape[0], self.size, ctx)
        ops.add_rms_norm_int8(stream.resid, stream.delta, self.weight, self.eps, out.codes, out.scales)
        if stream.delta is not None:
            stream.delta = stream.sumsq = None
        return out

    def lazy(self, stream: ResidualStream, ctx: StepContext) -> Int8Rows:
        return self.forward(stream, ctx)

    def forward_rows(self, stream, rows, num_rows, ctx):
        raise NotImplementedError("an 8-bit norm stands in front of a layer's projections, not in front of the output head")


@dataclass
class Int8KVCacheEntry:
    """The 8-bit cache of one call: codes ``[pages, kv_heads, page_size, head_dim]``, scales ``[pages, kv_heads]``."""

    group: int
    k: torch.Tensor
    v: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor
    page_size: int


@dataclass(frozen=True)
class Int8KVNeed(PagedNeed):
    """Pages of 8-bit keys and values with a 32-bit scale for every page and head. Storage ``[call, page, bytes of a page]``, as one
    run of bytes for each call: its key codes, its value codes, then the scales of both."""

    num_kv_heads: int
    head_dim: int
    window: int | None = None

    def bytes_per_token(self, element_size: int) -> int:
        # the scales of a page are 8 bytes a head: one byte a token and head with pages of 8 tokens (``bytes_per_page`` is exact)
        return self.num_kv_heads * (2 * self.head_dim + 1)

    def bytes_per_page(self, element_size: int, page_size: int) -> int:
        return 2 * self.num_kv_heads * page_size * self.head_dim + -(-2 * self.num_kv_heads * 4 // 16) * 16      # (calls start on 16 bytes)

    def allocate(self, num_calls, num_pages, page_size, dtype, device):
        if page_size * self.head_dim % 16:
            raise ValueError(f"pages of {page_size} tokens with heads of {self.head_dim}: 8-bit pages lie on 16 bytes")
        return torch.zeros((num_calls, num_pages, self.bytes_per_page(1, page_size)), dtype=torch.int8, device=device)

    def entry(self, storage, call_in_group, group, page_size):
        num_pages, heads = storage.shape[1], self.num_kv_heads
        codes = num_pages * heads * page_size * self.head_dim
        mine = storage[call_in_group].view(-1)
        k, v = (mine[i * codes: (i + 1) * codes].view(num_pages, heads, page_size, self.head_dim) for i in (0, 1))
        scales = mine[2 * codes: 2 * codes + 8 * num_pages * heads].view(torch.float32).view(2, num_pages, heads)
        return Int8KVCacheEntry(group, k, v, scales[0], scales[1], page_size)


_rows: dict[torch.device, list[torch.Tensor]] = {}


def _row_numbers(device: torch.device, t: int) -> torch.Tensor:
    """0, 1, 2, ... as int32: where each token's key and value lie in a scratch of one row per token. Recorded steps of any model
    hold the addresses of the numbers they were given, so numbers that were handed out are never let go of; new ones are at
    least twice as many, so all of them together are no more than twice the last. (A step runs before it is recorded: none
    are made inside a recording.)"""
    made = _rows.setdefault(device, [])
    if not made or made[-1].numel() < t:
        made.append(torch.arange(max(t, 2 * made[-1].numel() if made else 1 << 16), dtype=torch.int32, device=device))
    return made[-1][:t]


class Int8GQAAttention(GQAAttention):
    """``GQAAttention`` with 8-bit projections over an 8-bit cache. The new keys and values, normed and rotated in the model
    dtype, go through a scratch of one row per token into the cache's codes."""

    recordable = EVERY_STEP
    takes_lazy_input = False
    adds_to_stream = False

    def cache_need(self) -> Int8KVNeed:
        return Int8KVNeed(self.num_kv_heads, self.head_dim, self.window)

    def tensor_specs(self, prefix: str) -> list[TensorSpec]:
        return _projections_in_8_bits(super().tensor_specs(prefix))

    def bind(self, prefix: str, tensors: "Mapping[str, torch.Tensor | Int8Weight]") -> None:
        p = prefix + self.prefix
        self.qkv, self.o = Int8Weight.of(tensors[p + "qkv_proj.weight"]), Int8Weight.of(tensors[p + "o_proj.weight"])
        self.eight_bit = {p + "qkv_proj.weight": self.qkv, p + "o_proj.weight": self.o}
        if self.qk_norm:
            self.q_norm_w, self.k_norm_w = tensors[p + "q_norm.weight"], tensors[p + "k_norm.weight"]
        _row_numbers(self.qkv.codes.device, 1)

    def forward(self, x: Int8Rows, ctx: StepContext, cache: Int8KVCacheEntry, writes_cache: bool, position: Any) -> torch.Tensor:
        t, h, hkv, d = x.num_rows, self.num_heads, self.num_kv_heads, self.head_dim
        arena, group = ctx.arena, ctx.kv[cache.group]
        qkv = self.qkv.project(x, ctx, None if writes_cache else self.q_size)
        rot = None if position is None else position.qk_rotation()
        q, k, v = arena.take((t, h, d), ctx.dtype), arena.take((t, hkv, 1, d), ctx.dtype), arena.take((t, hkv, 1, d), ctx.dtype)
        ops.qk_norm_rope_write(qkv, q, self.q_norm_w, self.k_norm_w, self.qk_norm_eps, None if rot is None else rot.cos,
                               None if rot is None else rot.sin, 0 if rot is None else rot.rotary_dim,
                               False if rot is None else rot.interleaved, _row_numbers(qkv.device, t), k, v, 1, h, hkv, d, writes_cache)
        pages = (cache.k, cache.v, cache.k_scales, cache.v_scales, cache.page_size, group.block_tables, ctx)
        if writes_cache:
            ops.kv_write_int8(k.view(t, hkv, d), v.view(t, hkv, d), *pages)
        attn = arena.take((t, self.q_size), ctx.dtype)
        ops.paged_attention_int8(q, *pages, self.scale, self.window or 0, attn)
        rows = _take_rows(t, self.q_size, ctx)
        ops.act_mul_int8(attn, rows.codes, rows.scales, "none")
        return self.o.project(rows, ctx)


class Int8SwiGLU(SwiGLU):
    """``SwiGLU`` with 8-bit projections; the activation is 32-bit and rounded once, to the codes."""

    recordable = EVERY_STEP
    takes_lazy_input = False
    adds_to_stream = False

    def tensor_specs(self, prefix: str) -> list[TensorSpec]:
        return _projections_in_8_bits(super().tensor_specs(prefix))

    def bind(self, prefix: str, tensors: "Mapping[str, torch.Tensor | Int8Weight]") -> None:
        p = prefix + self.prefix
        self.gate_up, self.down = Int8Weight.of(tensors[p + "gate_up_proj.weight"]), Int8Weight.of(tensors[p + "down_proj.weight"])
        self.eight_bit = {p + "gate_up_proj.weight": self.gate_up, p + "down_proj.weight": self.down}

    def streamed_weights(self) -> list[torch.Tensor]:
        return []

    def forward(self, x: Int8Rows, ctx: StepContext) -> torch.Tensor:
        gate_up = self.gate_up.project(x, ctx)
        rows = _take_rows(x.num_rows, self.intermediate_size, ctx)
        ops.act_mul_int8(gate_up, rows.codes, rows.scales, "silu")
        return self.down.project(rows, ctx)


register_norm("rms_norm_int8", Int8RMSNorm)
register_mixer("gqa_attention_int8", Int8GQAAttention)
register_feed_forward("swiglu_int8", Int8SwiGLU)

# what stands for what, by the role's family of parts
_EIGHT_BIT = {"gqa_attention": "gqa_attention_int8", "swiglu": "swiglu_int8", "rms_norm": "rms_norm_int8"}


def eight_bit(spec: ModelSpec) -> ModelSpec:
    """The same model with its layers' projections, and the cache, in 8 bits. Embedding, final norm and output head stay."""
    def part(n: int, role: str, p: PartSpec) -> PartSpec:
        if p.kind not in _EIGHT_BIT or (p.kind == "rms_norm" and p.args.get("unit_offset")):
            raise UnsupportedConfigError(f"layer {n} of {spec.architecture}: no 8-bit form of {p.kind!r} ({role})")
        return PartSpec(_EIGHT_BIT[p.kind], p.args)

    layers = []
    for n, layer in enumerate(spec.layers):
        if layer.block != "prenorm" or "second_mixer" in layer.parts:
            raise UnsupportedConfigError(f"layer {n} of {spec.architecture}: no 8-bit form of its block {layer.block!r}")
        layers.append(replace(layer, parts={role: part(n, role, p) for role, p in layer.parts.items()}))
    return replace(spec, layers=tuple(layers))
