"""A full-attention layer's way from its activation to its output projection, on one GPU.

The reference's `encode_decode_full_layer` (src/metal_runtime.rs:1567-2020) without its norms and its output gate:

    q, k, v = projections(x)              one grouped launch, one activation read
    q = turned(q); cache <- turned(k), v  quantised as they are written
    a = attention(q, cache)               bf16
    out = output_projection(a)            fp32

`forward` enqueues five launches and allocates nothing, so that a step can be captured in a CUDA graph and replayed for every token: positions,
lengths and the page table are read on the device. torch is used for device buffers only.
"""
from __future__ import annotations

import torch

from . import capi
from .runtime import CudaRuntime, KvCache, KvTable, MappedQ4AffineJob, Q4RuntimeError

_POOLS = {"bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


class AttentionLayer:
    """`q`, `k`, `v`, `o`: jobs of the four projections (q: heads * head_dim outputs of `hidden` inputs, k and v: kv_heads * head_dim, o:
    `hidden` outputs of heads * head_dim inputs). `sequences` of up to `pages_per_sequence * page_tokens` tokens each; `forward` takes
    `tokens` (1...16) new ones of every sequence. Its buffers are on the runtime's device.

    The caller keeps up to date, on the device: `table` [sequences][pages_per_sequence] (numbers of the `pages` pages; each sequence has its
    own to begin with), `positions` [sequences * tokens] of the new tokens (negative: padded, for a sequence with fewer of them; they stand in
    front) and `lengths` [sequences], the new tokens counted in. `advance` does the last two."""

    def __init__(self, rt: CudaRuntime, q: MappedQ4AffineJob, k: MappedQ4AffineJob, v: MappedQ4AffineJob, o: MappedQ4AffineJob, hidden: int, heads: int,
                 kv_heads: int, head_dim: int, sequences: int, pages_per_sequence: int, page_tokens: int = 16, cache_format: str = "int8", rotary_dim: int = 64,
                 rotary_base: float = 1e7, rotary_scaling: dict | None = None, tokens: int = 1, scale: float | None = None, device: int | None = None):
        if device is None:
            device = rt.device
        if device != rt.device:
            raise Q4RuntimeError(13, f"buffers on device {device}, the runtime is on {rt.device}")
        for name, job, rows in (("q", q, heads * head_dim), ("k", k, kv_heads * head_dim), ("v", v, kv_heads * head_dim), ("o", o, hidden)):
            if job.output_rows != rows:
                raise Q4RuntimeError(6, f"{name} projection has {job.output_rows} elements, expected {rows}")
        if not 1 <= tokens <= 16:
            raise Q4RuntimeError(14, f"tokens {tokens} is not a number from 1 to 16")
        if sequences < 1 or pages_per_sequence < 1 or page_tokens < 16 or page_tokens % 16:
            raise Q4RuntimeError(13, "an attention layer needs sequences, pages and pages of a multiple of 16 tokens")
        if heads % kv_heads:
            raise Q4RuntimeError(6, f"heads has {heads} elements, expected a multiple of {kv_heads}")
        if cache_format not in _POOLS:
            raise Q4RuntimeError(13, f"unknown cache format {cache_format}")
        self.rt, self.q, self.k, self.v, self.o = rt, q, k, v, o
        self.hidden, self.heads, self.kv_heads, self.head_dim, self.tokens, self.sequences = hidden, heads, kv_heads, head_dim, tokens, sequences
        self.scale = head_dim ** -0.5 if scale is None else scale
        dev, pages, rows = torch.device("cuda", device), sequences * pages_per_sequence, sequences * tokens
        self.pools = [torch.zeros(pages, kv_heads, page_tokens, head_dim, dtype=_POOLS[cache_format], device=dev) for _ in range(2)]
        self.scales = None if cache_format == "bf16" else [torch.zeros(pages, kv_heads, page_tokens, device=dev) for _ in range(2)]
        self.table = torch.arange(pages, dtype=torch.int32, device=dev).view(sequences, pages_per_sequence)
        self.positions = torch.full((rows,), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=dev)
        self.queries, self.keys, self.values = (torch.empty(rows, n * head_dim, device=dev) for n in (heads, kv_heads, kv_heads))
        self.attended = torch.empty(rows, heads * head_dim, dtype=torch.bfloat16, device=dev)
        self.out = torch.empty(rows, hidden, device=dev)
        self.cache = KvCache(cache_format, kv_heads, head_dim, page_tokens, pages, self.pools[0].data_ptr(), self.pools[1].data_ptr(),
                             self.scales[0].data_ptr() if self.scales else 0, self.scales[1].data_ptr() if self.scales else 0)
        self.pages = KvTable(self.table.data_ptr(), sequences, pages_per_sequence)
        self.rotary = rt.rotary_create(rotary_dim, rotary_base, "half", rotary_scaling)

    def advance(self, new: torch.Tensor | None = None) -> None:
        """`new` [sequences] more tokens (`tokens` of each if None): sets `lengths` and `positions`, on torch's current stream."""
        self.lengths += self.tokens if new is None else new
        at = torch.arange(self.tokens, dtype=torch.int32, device=self.lengths.device) - self.tokens + self.lengths[:, None]
        if new is not None:
            at = torch.where(at >= (self.lengths - new)[:, None], at, -1)
        self.positions.copy_(at.reshape(-1))

    def forward(self, x_ptr: int, stream: int = 0) -> None:
        """x [sequences * tokens][hidden] bf16, row s * tokens + i for token i of sequence s; results in `out`. `stream` is ordered behind what
        set x, `table`, `positions` and `lengths`."""
        rt, rows, d, f32 = self.rt, self.sequences * self.tokens, self.head_dim, capi.Q4B_F32
        rt.matmul_batch_device(x_ptr, capi.Q4B_BF16, rows, self.hidden, [self.q, self.k, self.v], [t.data_ptr() for t in (self.queries, self.keys, self.values)], 0, stream)
        rt.rotary_device(self.rotary, self.queries.data_ptr(), f32, self.heads * d, rows, self.heads, d, self.positions.data_ptr(), self.queries.data_ptr(), f32, self.heads * d, stream)
        rt.kv_write_device(self.cache, self.pages, self.positions.data_ptr(), 0, rows, self.keys.data_ptr(), self.kv_heads * d, self.values.data_ptr(), self.kv_heads * d, f32,
                           self.rotary, stream)
        rt.attention_device(self.cache, self.pages, self.lengths.data_ptr(), self.queries.data_ptr(), f32, self.heads * d, self.heads, self.tokens, self.scale,
                            self.attended.data_ptr(), capi.Q4B_BF16, self.heads * d, stream)
        rt.matmul_batch_device(self.attended.data_ptr(), capi.Q4B_BF16, rows, self.heads * d, [self.o], [self.out.data_ptr()], 0, stream)

    def close(self) -> None:
        """Frees the rotary frequencies: graphs that have captured `forward` may not be replayed behind it, nor without the layer, whose
        buffers they use."""
        self.rotary.close()
