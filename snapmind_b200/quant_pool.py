"""A paged KV pool held in 8 bits: rows are quantised as they are written.

``QuantizedKVPool`` is :class:`snapmind_b200.paged_pool.PagedKVPool` with half the bytes
per token (of a 16-bit pool): the same block tables, reserve and release, ``append``,
``append_packed``, ``gather``, ``decode`` and ``attend_chunk``.

* ``k``, ``v``: ``torch.float8_e4m3fn`` ``[layer][block][head][slot][dim]``;
* ``scales``: uint8 ``[layer][block][head][2][slot]`` (K, V): exponent + 127 of a row.

A row x of one token and head is held as ``c * 2^e``: e the smallest integer in
[-100, 120] with ``max |x| <= 448 * 2^e``, c the e4m3 value nearest to ``x / 2^e`` (ties to
even).  So a value is off by at most 2^-4 of itself (or by 2^(e - 10), for values below
2^(e - 6)).  Infinities and NaN become NaN.  Queries, outputs and ``gather`` are in ``dtype``
(bf16, f16 or f32); attention takes the rows as they are held, also where ``dtype`` could not hold
them.  The reference cache has no 8-bit form.
"""
from __future__ import annotations

import torch

from snapmind_b200 import _lib
from snapmind_b200.paged_pool import PagedKVPool


class QuantizedKVPool(PagedKVPool):
    quantised = True

    def _allocate(self, shape) -> None:
        n_layers, num_blocks, heads, bs, _ = shape
        self._pool_code = _lib.DTYPE_E4M3
        self.k = torch.empty(shape, dtype=torch.float8_e4m3fn, device=self.device)
        self.v = torch.empty(shape, dtype=torch.float8_e4m3fn, device=self.device)
        self.scales = torch.empty((n_layers, num_blocks, heads, 2, bs), dtype=torch.uint8, device=self.device)
        self.scale_layer_stride = num_blocks * heads * 2 * bs
        self._values = torch.empty(0, dtype=self.dtype, device=self.device)  # of the type that is read back

    def append(self, layer: int | None, k_new: torch.Tensor, v_new: torch.Tensor, slot_starts=None,
               slot_start0: int | None = None) -> None:
        """``PagedKVPool.append``, quantising: ``[B, H, D]``, ``[B, H, T, D]`` or, with
        ``layer=None``, ``[L, B, H, T, D]`` rows of any float dtype."""
        if k_new.dim() == 3:
            k_new, v_new = k_new.unsqueeze(2), v_new.unsqueeze(2)
        if k_new.dim() == 4:
            if layer is None:
                raise ValueError("layer is required for [B, H, T, D] inputs")
            k_new, v_new = k_new.unsqueeze(0), v_new.unsqueeze(0)
        n_layers, batch, _, n_tokens, _ = k_new.shape
        starts, start0 = self._slot_args(n_tokens, slot_starts, slot_start0)
        self._append_chunk(0 if layer is None else layer, k_new, v_new, (0, 2, 3), 1, None, n_layers, batch, n_tokens,
                           batch * n_tokens, starts, start0)

    def gather(self, batch: int | None = None, layers: range | None = None, out=None):
        """``PagedKVPool.gather``, read back to ``dtype`` (values past its largest are held to it)."""
        batch = self.max_seqs if batch is None else batch
        if not 0 <= batch <= self.max_seqs:
            raise ValueError(f"gather: {batch} sequences, the pool holds {self.max_seqs}")
        layers = range(self.n_layers) if layers is None else layers
        total = int(self._host_lens[:batch].sum())
        per_layer = total * self.n_kv_heads * self.head_dim
        if out is None:
            k_out, v_out = self._values.new_empty((len(layers), per_layer)), self._values.new_empty((len(layers), per_layer))
        else:
            k_out, v_out = out
            for t in (k_out, v_out):
                if (t.dtype != self.dtype or t.dim() != 2 or t.shape[0] < len(layers) or t.shape[1] != k_out.shape[1]
                        or t.shape[1] < per_layer or not t.is_contiguous()):
                    raise ValueError("gather output too small or not contiguous")
        if per_layer == 0 or len(layers) == 0:
            return k_out, v_out
        if layers.step != 1 or not 0 <= layers.start <= layers.stop <= self.n_layers:
            raise ValueError(f"gather: {layers} of a pool of {self.n_layers} layers")
        _lib.require_same("gather", self.block_tables, k_out, v_out)
        first = layers.start * self.layer_stride
        with self._on_device():
            status = _lib.load().snapmind_kv_gather_quant(
                self.k.data_ptr() + first, self.v.data_ptr() + first,
                self.scales.data_ptr() + layers.start * self.scale_layer_stride, self.layer_stride,
                self.scale_layer_stride, k_out.data_ptr(), v_out.data_ptr(), self._dcode, k_out.shape[1],
                k_out.shape[1], self.block_tables.data_ptr(), self.max_blocks_per_seq, self.max_blocks_per_seq,
                self.seq_lens.data_ptr(), len(layers), batch, self.n_kv_heads, self.head_dim, self.block_size,
                self.num_blocks, self.err.data_ptr(), _lib.raw_stream(self._index),
            )  # fmt: skip
        if status:
            _lib.check(status, "QuantizedKVPool.gather")
        return k_out, v_out

    def decode(self, layer: int, q: torch.Tensor, out: torch.Tensor | None = None, scale: float | None = None,
               batch: int | None = None, split_tokens: int = 0, force_generic: bool = False,
               max_seq_len: int | None = None, peers=None, append=None, window: int = 0,
               sinks: int = 0) -> torch.Tensor:
        """``PagedKVPool.decode`` over the 8-bit rows (``split_tokens`` and ``max_seq_len``
        have no use: the kernel plans from the device lengths)."""
        if peers is not None:
            raise ValueError("QuantizedKVPool: decode has no peer form")
        return self._attend_tokens(layer, q, out, scale, batch, window, sinks, force_generic, append)

    def decode_layers(self, *args, **kwargs):
        raise NotImplementedError("QuantizedKVPool: decode one layer at a time")

    def attend_causal(self, layer: int, b: int, q: torch.Tensor, out: torch.Tensor, n_b: int,
                      scale: float | None = None) -> torch.Tensor:
        """``PagedKVPool.attend_causal`` (``q``/``out`` ``[Hq, T, D]``, the sequence's first ``n_b`` tokens, the
        newest T of them the queries') as a chunk of one sequence."""
        n_t = q.shape[1]
        if n_t == 0:
            return out
        if n_b < n_t:
            raise ValueError(f"attend_causal: {n_t} queries of {n_b} tokens")
        cu = torch.zeros(2, dtype=torch.int32, device=self.device)
        cu[1] = n_t
        row = self.block_tables[b].data_ptr(), self._lens_ladder(n_b).data_ptr() + 4 * (n_b - 1)
        self._attend(layer, q.transpose(0, 1), cu, out.transpose(0, 1), scale, 0, 0, 0, row=row)
        return out
