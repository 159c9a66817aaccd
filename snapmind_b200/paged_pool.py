"""Many sequences on one paged KV pool — the batched form of PagedKVCache.

The reference cache holds one sequence per instance (snapmind/kv_cache/paged.py:51-52
reads ``key[0]`` only).  Serving many sequences needs the same slot arithmetic
over one shared pool; this class is that extension, with all state on the GPU:

* ``k``, ``v``: ``[layer][block][head][slot][dim]``; a block id is valid in every
  layer, so one block table row per sequence serves all layers;
* ``block_tables`` int32 ``[max_seqs][max_blocks_per_seq]``, ``seq_lens`` int32;
* a device free stack (``free_stack``, ``free_top``) from which
  ``snapmind_kv_reserve`` grows tables deterministically (ascending sequence
  order, blocks from the top of the stack);
* with ``mass=True`` also ``mass``, f32 ``[layer][block][head][slot]``: the attention weight
  that each cached token got from the calls with ``accumulate=True`` (zero when ``reserve``
  makes room for it), by which ``evict`` thins the sequences.

Block bookkeeping (tables, lengths, free stack, reserve/release) is in
:class:`snapmind_b200.block_pool.BlockPool`.
"""
from __future__ import annotations

from collections.abc import MutableMapping

import numpy as np
import torch

from snapmind_b200 import _lib
from snapmind_b200.block_pool import BlockPool


_FAR = 1 << 30  # no position is as far


def _share(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.untyped_storage().data_ptr() == b.untyped_storage().data_ptr()


class PagedKVPool(BlockPool):
    quantised = False  # pool elements are the values themselves

    def __init__(
        self,
        n_layers: int,
        n_kv_heads: int,
        head_dim: int,
        num_blocks: int,
        max_seqs: int,
        max_blocks_per_seq: int,
        block_size: int = 16,
        dtype: torch.dtype = torch.bfloat16,
        device: torch.device | str | None = None,
        mass: bool = False,
    ):
        super().__init__(num_blocks, max_seqs, max_blocks_per_seq, block_size, device)
        self.n_layers, self.n_kv_heads, self.head_dim = n_layers, n_kv_heads, head_dim
        self.dtype = dtype
        self._dcode = _lib.dtype_code(dtype)
        self.layer_stride = num_blocks * n_kv_heads * block_size * head_dim
        self.scale_layer_stride = 0
        self._allocate((n_layers, num_blocks, n_kv_heads, block_size, head_dim))
        # attention weight that every cached token got so far, of the layer and kv head, in the pool's own layout
        self.mass = None
        if mass:
            self.mass = torch.zeros((n_layers, num_blocks, n_kv_heads, block_size), dtype=torch.float32, device=self.device)
            self._reserve_status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._workspace = _lib.DecodeWorkspace(self.device)
        with self._on_device():
            self._chunk_ws = _lib.load().snapmind_paged_gqa_chunk_workspace_bytes(head_dim)

    def _allocate(self, shape) -> None:
        self._pool_code = self._dcode
        self.k = torch.empty(shape, dtype=self.dtype, device=self.device)
        self.v = torch.empty(shape, dtype=self.dtype, device=self.device)

    def append(self, layer: int | None, k_new: torch.Tensor, v_new: torch.Tensor, slot_starts=None,
               slot_start0: int | None = None) -> None:
        """Write new tokens' K/V rows.

        ``k_new``: ``[B, H, D]`` (one token, layer ``layer``), ``[B, H, T, D]``,
        or ``[L, B, H, T, D]`` with ``layer=None`` (all layers at once).  By
        default token t of sequence b goes to slot ``seq_lens[b] - T + t`` — the
        slots that the last ``reserve(T)`` added.
        """
        if k_new.dim() == 3:
            k_new, v_new = k_new.unsqueeze(2), v_new.unsqueeze(2)
        if k_new.dim() == 4:
            if layer is None:
                raise ValueError("layer is required for [B, H, T, D] inputs")
            k_new, v_new = k_new.unsqueeze(0), v_new.unsqueeze(0)
            n_layers, base = 1, layer
        else:
            n_layers, base = k_new.shape[0], (0 if layer is None else layer)
        if k_new.shape != v_new.shape or k_new.dtype != v_new.dtype:
            raise ValueError("append: k and v rows differ in shape or dtype")
        _lib.require_same("append", self.block_tables, k_new, v_new)
        if k_new.stride() != v_new.stride() or k_new.stride(-1) != 1:
            k_new, v_new = k_new.contiguous(), v_new.contiguous()
        _, batch, n_heads, n_tokens, head_dim = k_new.shape
        if n_heads != self.n_kv_heads or head_dim != self.head_dim:
            raise ValueError(f"expected {self.n_kv_heads} heads of {self.head_dim}, got {tuple(k_new.shape)}")
        starts_ptr, start0 = self._slot_args(n_tokens, slot_starts, slot_start0)
        st = k_new.stride()
        status = _lib.load().snapmind_kv_append(
            self.k[base].data_ptr(), self.v[base].data_ptr(), self._dcode, self.layer_stride,
            k_new.data_ptr(), v_new.data_ptr(), _lib.dtype_code(k_new.dtype),
            st[0], st[1], st[2], st[3],
            self.block_tables.data_ptr(), self.max_blocks_per_seq, 0, self.max_blocks_per_seq,
            starts_ptr, start0,
            n_layers, batch, n_tokens, n_heads, head_dim, self.block_size, self.num_blocks,
            self.err.data_ptr(), self._stream(),
        )  # fmt: skip
        _lib.check(status, "PagedKVPool.append")

    def append_rope(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor,
                    sin: torch.Tensor, positions: torch.Tensor, cu_new: torch.Tensor | None = None,
                    q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-6,
                    out: torch.Tensor | None = None) -> torch.Tensor:
        """Norm, rotate and store new tokens in one pass: returns the rotated queries.

        ``q`` ``[total, Hq, D]``, ``k``/``v`` ``[total, H, D]``, one dtype (any float dtype, ``out`` has it too).
        Queries and keys are normalised per head, ``x / sqrt(mean x^2 + eps) * norm`` (``q_norm`` / ``k_norm``:
        ``[D]``, or ``[heads, D]`` with weights for each head; ``None``: as they are), and rotated by the rows of ``cos`` /
        ``sin`` (f32 ``[n_pos, R]``, rotate-half over the first R dims) at ``positions`` (int64 ``[total]``): the tokens'
        own, which their indexes in a cache that evicts are not.  All in f32, rounded once.  K and V go where
        ``append_packed`` puts them (``cu_new`` ``[B + 1]``), or without ``cu_new`` token b is the newest of
        sequence b.  ``out`` may be ``q``.  A position outside the tables leaves its token out (``check()`` raises)."""
        total, n_q, d = q.shape
        want = (total, self.n_kv_heads, self.head_dim)
        if d != self.head_dim or k.shape != want or v.shape != want:
            raise ValueError(f"append_rope: expected q [total, heads, {self.head_dim}] and k, v {list(want)}, got "
                             f"{tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
        dtype = q.dtype
        if k.dtype != dtype or v.dtype != dtype:
            raise TypeError("append_rope: q, k and v differ in dtype")
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer {layer} of a pool of {self.n_layers}")
        batch, cu = total, None
        if cu_new is not None:
            _lib.require_offsets("append_rope", cu_new, self.block_tables)
            batch, cu = cu_new.shape[0] - 1, cu_new.data_ptr()
        if batch > self.max_seqs:
            raise ValueError(f"append_rope: {batch} sequences, the pool holds {self.max_seqs}")
        if positions.dtype != torch.int64 or positions.shape != (total,):
            raise ValueError(f"append_rope: positions must be int64 [{total}]")
        q_st, k_st, v_st = q.stride(), k.stride(), v.stride()
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            o_st = out.stride()
        else:
            o_st = out.stride()
            if out.shape != q.shape or out.dtype != dtype or o_st[2] != 1:
                raise ValueError("append_rope: out must have q's shape and dtype, head dim contiguous")
        _lib.require_same("append_rope", self.block_tables, q, k, v, cos, sin, positions, out)
        rot, qn_st, kn_st = _lib.rope_args("append_rope", q, cos, sin, q_norm, k_norm, n_q, self.n_kv_heads, eps)
        if q_st[2] != 1 or k_st[2] != 1 or v_st[2] != 1:
            q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
            q_st, k_st, v_st = q.stride(), k.stride(), v.stride()
        if total > 1 and positions.stride(0) != 1:
            positions = positions.contiguous()
        step = layer * self.layer_stride * self.k.element_size()
        tables = self.block_tables.data_ptr()
        with self._on_device():
            status = _lib.load().snapmind_norm_rope_append(
                q.data_ptr(), q_st[0], q_st[1], out.data_ptr(), o_st[0], o_st[1], n_q,
                k.data_ptr(), k_st[0], k_st[1], v.data_ptr(), v_st[0], v_st[1], _lib.dtype_code(dtype),
                _lib.ptr(q_norm), qn_st, _lib.ptr(k_norm), kn_st, eps, cos.data_ptr(), sin.data_ptr(), rot, cos.shape[0],
                positions.data_ptr(), self.k.data_ptr() + step, self.v.data_ptr() + step,
                self.scales.data_ptr() + layer * self.scale_layer_stride if self.quantised else None, self._pool_code,
                tables, self.max_blocks_per_seq, self.max_blocks_per_seq, self.seq_lens.data_ptr(),
                cu, batch, total, self.n_kv_heads, d, self.block_size, self.num_blocks, self.err.data_ptr(),
                _lib.raw_stream(self._index),
            )  # fmt: skip
        if status:
            _lib.check(status, f"{type(self).__name__}.append_rope")
        return out

    def append_packed(self, layer: int | None, k_new: torch.Tensor, v_new: torch.Tensor,
                      cu_new: torch.Tensor) -> None:
        """Write the K/V rows of a ragged chunk, the ones that the last ``reserve_each``
        made room for.

        ``k_new``: ``[total, H, D]`` (layer ``layer``) or ``[L, total, H, D]``
        (``layer=None``: layers 0 .. L-1); ``cu_new`` int32 ``[B + 1]`` on the device: sequence
        b owns rows ``cu_new[b] .. cu_new[b + 1] - 1``, its newest tokens.
        """
        _lib.require_offsets("append", cu_new, self.block_tables)
        if k_new.dim() == 3:
            if layer is None:
                raise ValueError("layer is required for [total, H, D] inputs")
            k_new, v_new = k_new.unsqueeze(0), v_new.unsqueeze(0)
        n_layers, total = k_new.shape[:2]
        self._append_chunk(0 if layer is None else layer, k_new, v_new, (0, 2, 1), None, cu_new, n_layers,
                           cu_new.shape[0] - 1, 0, total, self.seq_lens.data_ptr(), 0)

    def _append_chunk(self, base, k_new, v_new, axes, seq_axis, cu, n_layers, batch, n_tokens, total, starts, start0):
        """``axes``: where the layer, head and token axes are; ``seq_axis``: the sequence axis or None."""
        _lib.require_same("append", self.block_tables, k_new, v_new)
        shape = k_new.shape
        if shape != v_new.shape or k_new.dtype != v_new.dtype:
            raise ValueError("append: k and v rows differ in shape or dtype")
        if len(shape) < 4 or shape[axes[1]] != self.n_kv_heads or shape[-1] != self.head_dim:
            raise ValueError(f"expected {self.n_kv_heads} heads of {self.head_dim}, got {tuple(shape)}")
        if not 0 <= base <= self.n_layers - n_layers:
            raise ValueError(f"append: layers {base} .. {base + n_layers - 1} of a pool of {self.n_layers}")
        if batch > self.max_seqs or batch < 0:
            raise ValueError(f"append: {batch} sequences, the pool holds {self.max_seqs}")
        st = k_new.stride()
        if st != v_new.stride() or st[-1] != 1:
            k_new, v_new = k_new.contiguous(), v_new.contiguous()
            st = k_new.stride()
        row = self.layer_stride * self.k.element_size()
        scales = self.scales.data_ptr() + base * self.scale_layer_stride if self.quantised else None
        with self._on_device():
            status = _lib.load().snapmind_kv_append_chunk(
                self.k.data_ptr() + base * row, self.v.data_ptr() + base * row, scales, self._pool_code,
                self.layer_stride, self.scale_layer_stride, k_new.data_ptr(), v_new.data_ptr(),
                _lib.dtype_code(k_new.dtype), st[axes[0]], 0 if seq_axis is None else st[seq_axis], st[axes[1]],
                st[axes[2]], self.block_tables.data_ptr(), self.max_blocks_per_seq, self.max_blocks_per_seq,
                starts, start0, None if cu is None else cu.data_ptr(), n_layers, batch, n_tokens, total,
                self.n_kv_heads, self.head_dim, self.block_size, self.num_blocks, self.err.data_ptr(), _lib.raw_stream(self._index),
            )  # fmt: skip
        if status:
            _lib.check(status, f"{type(self).__name__}.append")

    # -------------------------------------------------------------- eviction
    def _reserved(self, n_new, batch, counts=None):
        if self.mass is None or n_new == 0:
            return
        with self._on_device():
            status = _lib.load().snapmind_kv_clear_mass(
                self.mass.data_ptr(), self.mass.stride(0), self.block_tables.data_ptr(), self.max_blocks_per_seq,
                self.max_blocks_per_seq, self.seq_lens.data_ptr(), _lib.ptr(counts), n_new, batch, self.n_layers,
                self.n_kv_heads, self.block_size, self.num_blocks, _lib.ptr(self._reserve_status), _lib.raw_stream(self._index),
            )  # fmt: skip
        _lib.check(status, f"{type(self).__name__}.reserve")

    def set_state(self, tables, lens, free_stack) -> None:
        super().set_state(tables, lens, free_stack)
        if self.mass is not None:
            self.mass.zero_()

    def evict(self, budget: int, recent: int = 0, sinks: int = 0, batch: int | None = None, seqs=None,
              into=None) -> torch.Tensor:
        """Thin sequences to ``budget`` tokens by ``mass``: each layer and kv head keeps the first ``sinks``
        tokens, the newest ``recent``, and of the others those with the largest accumulated weight (equal ones: the lowest
        index; a NaN counts as the largest).  What stays moves to the front in its order, with its mass; a sequence of
        at most ``budget`` tokens stays as it is.  The lengths of a sequence are those of all its layers and heads, so all
        are thinned alike.  Keys keep the rotation they were stored with.

        The first ``batch`` sequences, or those named in ``seqs`` (distinct), lose their last blocks to the free
        stack.  With ``into`` (as many distinct sequences, none of them in ``seqs``) they stay whole, and what the
        targets held is replaced by the thinned copies.  Sequences must not share blocks.

        Returns the kept indexes, int32 ``[n_layers, n, n_kv_heads, budget]``, ascending, -1 behind the last."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("evict: a captured step takes evict_device, and the host's lengths by account_evict")
        if seqs is not None and batch is not None:
            raise ValueError("evict: batch or seqs, not both")
        if into is not None and seqs is None:
            raise ValueError("evict: into goes with seqs")
        ids = np.arange(self.max_seqs if batch is None else batch) if seqs is None else np.asarray(seqs, dtype=np.int64).reshape(-1)
        to = ids if into is None else np.asarray(into, dtype=np.int64).reshape(-1)
        every = ids if into is None else np.concatenate([ids, to])
        if len(to) != len(ids) or len(np.unique(every)) != len(every) or (every.size and not 0 <= every.min() <= every.max() < self.max_seqs):
            raise ValueError("evict: sequences must be distinct and inside the pool, and each have a target of its own")
        if budget < 1:
            raise ValueError(f"evict: a budget of {budget}")
        lens = self._host_lens[ids]
        ends, held = np.minimum(lens, budget), self._host_lens[to]
        grow = (ends + self.block_size - 1) // self.block_size - (held + self.block_size - 1) // self.block_size
        if into is not None and int(np.maximum(grow, 0).sum()) > self._host_free:
            raise RuntimeError(_lib.OUT_OF_BLOCKS_MSG)
        named = [None, None]
        if seqs is not None:  # pinned, so that the copy waits for nothing
            both = torch.from_numpy((ids if into is None else every).astype(np.int32)).pin_memory().to(self.device, non_blocking=True)
            named = [both[:len(ids)], None if into is None else both[len(ids):]]
        kept = self._evict(budget, recent, sinks, len(ids), *named, int(lens.max()) if lens.size else 1)
        self._host_lens[to] = ends
        self._host_free -= int(grow.sum())
        return kept

    def evict_device(self, budget: int, recent: int = 0, sinks: int = 0, batch: int | None = None) -> torch.Tensor:
        """The device part of ``evict`` in place for the first ``batch`` sequences: launches that a CUDA graph can replay.
        The caller accounts every replay with ``account_evict``."""
        return self._evict(budget, recent, sinks, self.max_seqs if batch is None else batch, None, None, 0)

    def account_evict(self, budget: int, batch: int | None = None) -> None:
        """Bring the host mirrors to what ``evict(budget, batch=batch)`` makes of them."""
        lens = self._host_lens[:self.max_seqs if batch is None else batch]
        ends = np.minimum(lens, budget)
        self._host_free += int(((lens + self.block_size - 1) // self.block_size - (ends + self.block_size - 1) // self.block_size).sum())
        lens[:] = ends

    def _evict(self, budget, recent, sinks, n, ids, to, max_len):
        if self.mass is None:
            raise ValueError("evict needs a pool with mass=True")
        if budget < 1 or recent < 0 or sinks < 0 or recent + sinks > budget:
            raise ValueError(f"evict: the newest {recent} and the first {sinks} tokens do not fit a budget of {budget}")
        if not 0 <= n <= self.max_seqs:
            raise ValueError(f"evict: {n} sequences, the pool holds {self.max_seqs}")
        kept = torch.empty((self.n_layers, n, self.n_kv_heads, budget), dtype=torch.int32, device=self.device)
        with self._on_device():
            status = _lib.load().snapmind_kv_evict_by_mass(
                self.k.data_ptr(), self.v.data_ptr(), self.scales.data_ptr() if self.quantised else None, self._pool_code,
                self.layer_stride, self.scale_layer_stride, self.mass.data_ptr(), self.mass.stride(0),
                self.block_tables.data_ptr(), self.max_blocks_per_seq, self.max_blocks_per_seq, self.seq_lens.data_ptr(),
                _lib.ptr(ids), _lib.ptr(to), n, budget, recent, sinks, max_len, kept.data_ptr(), self.free_stack.data_ptr(),
                self.free_top.data_ptr(), self.n_layers, self.n_kv_heads, self.head_dim, self.block_size, self.num_blocks,
                self.err.data_ptr(), _lib.raw_stream(self._index),
            )  # fmt: skip
        if status:
            _lib.check(status, f"{type(self).__name__}.evict")
        return kept

    # ----------------------------------------------------------------- reads
    def attend_chunk(self, layer: int, q: torch.Tensor, cu_q: torch.Tensor, out: torch.Tensor | None = None,
                     scale: float | None = None, window: int = 0, sinks: int = 0,
                     force_generic: bool = False, accumulate: bool = False) -> torch.Tensor:
        """Causal attention of a ragged chunk of new tokens against layer ``layer``, in
        one launch: pieces of prompts, drafted tokens and single tokens together.

        ``q``/``out``: ``[total, Hq, D]``; ``cu_q`` int32 ``[B + 1]`` on the device: sequence
        b's new tokens are rows ``cu_q[b] .. cu_q[b + 1] - 1`` (none when equal), already
        stored in the pool as its newest.  With ``window`` > 0 a query sees the
        ``window`` positions up to its own and the first ``sinks``.  Rows of ``out`` that
        belong to no sequence are left as they were (whatever a new ``out`` holds).

        A position that a query does not see never counts, whatever K and V hold there (a NaN in V
        of one of the chunk's tokens reaches the queries from it on).  ``force_generic`` takes the
        CUDA-core kernel, all in f32.

        ``accumulate`` adds to ``mass[layer]`` the weight that each cached token gets from the chunk's queries, summed over
        them and over the query heads that share its kv head (in f32, the same bits every time).  Such calls of one
        layer must not overlap on the GPU, and the sequences must not share blocks."""
        _lib.require_offsets("attend_chunk", cu_q, self.block_tables)
        if cu_q.shape[0] - 1 > self.max_seqs:
            raise ValueError(f"attend_chunk: {cu_q.shape[0] - 1} sequences, the pool holds {self.max_seqs}")
        return self._attend(layer, q, cu_q, out, scale, window, sinks,
                            _lib.DECODE_FORCE_GENERIC if force_generic else 0, accumulate=accumulate)

    def _attend_tokens(self, layer, q, out, scale, batch, window, sinks, force_generic, append, accumulate=False):
        """One query per sequence for the first ``batch`` sequences, their newest token stored first if given."""
        rows = out
        if batch is not None:
            if not 0 <= batch <= q.shape[0]:
                raise ValueError(f"decode: batch {batch} of {q.shape[0]} queries")
            q, rows = q[:batch], None if out is None else out[:batch]
        if append is not None:
            want = (q.shape[0], self.n_kv_heads, self.head_dim)
            if append[0].shape != want or append[1].shape != want:
                raise ValueError(f"append rows must be {list(want)}, got {tuple(append[0].shape)} and {tuple(append[1].shape)}")
        got = self._attend(layer, q, None, rows, scale, window, sinks,
                           _lib.DECODE_FORCE_GENERIC if force_generic else 0, append, accumulate=accumulate)
        return got if out is None else out

    def _attend(self, layer, q, cu, out, scale, window, sinks, flags, append=None, row=None, accumulate=False):
        """``row``: ``(table, length)`` pointers of the one sequence, in place of the pool's own tables and lengths."""
        total, n_q, d = q.shape
        if q.dtype != self.dtype:
            raise TypeError(f"q dtype {q.dtype} != pool dtype {self.dtype}")
        if d != self.head_dim:
            raise ValueError(f"q head dim {d} != the pool's {self.head_dim}")
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer {layer} of a pool of {self.n_layers}")
        if cu is None and total > self.max_seqs:
            raise ValueError(f"decode: {total} sequences, the pool holds {self.max_seqs}")
        if accumulate and self.mass is None:
            raise ValueError("accumulate needs a pool with mass=True")
        q_st = q.stride()
        if q_st[2] != 1:
            q = q.contiguous()
            q_st = q.stride()
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            o_st = out.stride()
        else:
            o_st = out.stride()
            if out.shape != q.shape or out.dtype != self.dtype or o_st[2] != 1:
                raise ValueError("out must have q's shape and dtype, head dim contiguous")
            if (accumulate or (self.quantised and self.dtype == torch.float16)) and _share(q, out):
                q = q.clone()  # such a call may be done over, or takes the scores anew, with the queries it began with
                q_st = q.stride()
        if q.device != self._device or out.device != self._device:
            _lib.require_same("attend", self.block_tables, q, out)
        if append is not None:
            self.append(layer, *append)
        if not (-1 <= window <= _FAR and -1 <= sinks <= _FAR):  # the C entry takes 32 bits
            window, sinks = (max(-1, min(x, _FAR)) for x in (window, sinks))
        lib = _lib.load()
        # a workspace of its own for every call: calls on several streams, or in several
        # captured graphs, never share one
        need, mass = self._chunk_ws, None
        if accumulate:
            # a decode on the tensor cores keeps its scores: room for what its sequences, or the pool, can hold
            keeps = cu is None and self.dtype != torch.float32 and not flags and (self.block_size in (16, 32) or self.block_size % 64 == 0)
            need = lib.snapmind_paged_gqa_chunk_mass_workspace_bytes(d, total, n_q, self.n_kv_heads, self.block_size,
                                                                     min(self.num_blocks, max(1, total * self.max_blocks_per_seq)), keeps)
            mass = self.mass.data_ptr() + 4 * layer * self.num_blocks * self.n_kv_heads * self.block_size
        ws = torch.empty(need, dtype=torch.uint8, device=self._device)
        step = layer * self.layer_stride * self.k.element_size()
        scales = self.scales.data_ptr() + layer * self.scale_layer_stride if self.quantised else None
        with self._on_device():
            status = lib.snapmind_paged_gqa_chunk_mass(
                q.data_ptr(), q_st[0], q_st[1], self._dcode, self.k.data_ptr() + step,
                self.v.data_ptr() + step, scales, self._pool_code,
                self.block_tables.data_ptr() if row is None else row[0],
                self.max_blocks_per_seq, self.max_blocks_per_seq, self.seq_lens.data_ptr() if row is None else row[1],
                None if cu is None else cu.data_ptr(), out.data_ptr(), o_st[0], o_st[1],
                d ** -0.5 if scale is None else scale, total if cu is None else cu.shape[0] - 1, total, n_q,
                self.n_kv_heads, d, self.block_size, self.num_blocks, window, sinks, flags, mass, ws.data_ptr(), need,
                self.err.data_ptr(), _lib.raw_stream(self._index),
            )  # fmt: skip
        if status:
            _lib.check(status, f"{type(self).__name__}.attend")
        return out

    def gather(self, batch: int | None = None, layers: range | None = None, out=None):
        """Packed K/V of the first ``batch`` sequences.

        Returns ``(k, v)`` of shape ``[n_layers, total_tokens * H * D]`` where the
        row of each layer is the concatenation over b of ``(H, len_b, D)`` — for
        one sequence the tensor ``PagedKVCache.fetch`` returns.
        """
        batch = self.max_seqs if batch is None else batch
        layers = range(self.n_layers) if layers is None else layers
        total = int(self._host_lens[:batch].sum())
        per_layer = total * self.n_kv_heads * self.head_dim
        if out is None:
            k_out = torch.empty((len(layers), per_layer), dtype=self.dtype, device=self.device)
            v_out = torch.empty_like(k_out)
        else:
            k_out, v_out = out
            for t in (k_out, v_out):
                if t.dtype != self.dtype or t.shape[0] < len(layers) or t[0].numel() < per_layer or not t.is_contiguous():
                    raise ValueError("gather output too small or not contiguous")
        if per_layer == 0 or len(layers) == 0:
            return k_out, v_out
        status = _lib.load().snapmind_kv_gather(
            self.k[layers.start].data_ptr(), self.v[layers.start].data_ptr(), self._dcode, self.layer_stride,
            k_out.data_ptr(), v_out.data_ptr(), per_layer, per_layer,
            self.block_tables.data_ptr(), self.max_blocks_per_seq, 0, self.max_blocks_per_seq,
            self.seq_lens.data_ptr(), 0,
            len(layers), batch, self.n_kv_heads, self.head_dim, self.block_size, self.num_blocks,
            self.err.data_ptr(), self._stream(),
        )  # fmt: skip
        _lib.check(status, "PagedKVPool.gather")
        return k_out, v_out

    def _decode_workspace(self, batch, n_q_heads, max_len, split):
        lib = _lib.load()
        need = lib.snapmind_paged_gqa_decode_workspace_bytes(
            batch, n_q_heads, self.n_kv_heads, self.head_dim, max_len, split
        )
        return self._workspace.get(batch, self.n_kv_heads, need)

    def decode_layers(self, q: torch.Tensor, out: torch.Tensor | None = None, scale: float | None = None,
                      split_tokens: int = 0, max_seq_len: int | None = None, peers=None) -> torch.Tensor | None:
        """Paged GQA decode of layers 0 .. L-1 in one launch: ``q`` ``[L, B, Hq, D]`` ->
        ``[L, B, Hq, D]``.

        The pool is layer-contiguous, so block ``p`` of layer ``l`` is block
        ``l * num_blocks + p`` of one pool spanning every layer; launch row
        ``l * B + b`` is sequence ``b`` of layer ``l``, its table row shifted by
        ``l * num_blocks`` (entries outside ``[0, num_blocks)`` stay invalid, so the
        kernel still flags them).  ``q`` (and ``out``) must step uniformly over
        (layer, sequence) rows: ``stride(0) == B * stride(1)``.  ``peers`` as in
        ``decode``, with ``out_stride_seq`` the row stride of every rank's
        ``[L, B, Hq, D]`` receive region."""
        n_l, batch, n_q, d = q.shape
        if n_l > self.k.shape[0]:
            raise ValueError(f"{n_l} layers > the pool's {self.k.shape[0]}")
        if q.dtype != self.dtype or q.stride(-1) != 1 or q.stride(0) != batch * q.stride(1):
            raise ValueError("q must be [L, B, Hq, D] in the pool's dtype with uniformly strided rows")
        if out is None and peers is None:
            out = torch.empty((n_l, batch, n_q, d), dtype=self.dtype, device=self.device)
        if out is not None and (out.stride(-1) != 1 or out.stride(0) != batch * out.stride(1)):
            raise ValueError("out must be [L, B, Hq, D] with uniformly strided rows")
        scale = self.head_dim ** -0.5 if scale is None else scale
        if max_seq_len is None:
            max_seq_len = max(1, int(self._host_lens[:batch].max())) if batch else 1
        rows = n_l * batch
        lib = _lib.load()
        split = split_tokens or lib.snapmind_paged_gqa_decode_split_tokens(rows, self.n_kv_heads, max_seq_len,
                                                                           self.block_size)
        ws = self._decode_workspace(rows, n_q, max_seq_len, split)
        t = self.block_tables[:batch]
        offs = torch.arange(n_l, dtype=torch.int32, device=self.device).view(n_l, 1, 1) * self.num_blocks
        tables = torch.where((t >= 0) & (t < self.num_blocks), t.unsqueeze(0) + offs, torch.full_like(t, -1))
        lens = self.seq_lens[:batch].unsqueeze(0).expand(n_l, batch).contiguous()
        span = n_l * self.num_blocks
        if peers is not None:
            status = lib.snapmind_paged_gqa_decode_peers(
                q.data_ptr(), q.stride(1), q.stride(2), self.k.data_ptr(), self.v.data_ptr(), self._dcode,
                tables.data_ptr(), self.max_blocks_per_seq, self.max_blocks_per_seq, lens.data_ptr(), None,
                peers.out_ptrs.data_ptr(), peers.n, peers.head_offset, peers.out_stride_seq, peers.out_stride_head,
                float(scale), rows, n_q, self.n_kv_heads, self.head_dim, self.block_size, span,
                max_seq_len, split, 0, ws.data_ptr(), ws.numel(), self.err.data_ptr(), self._stream(),
            )  # fmt: skip
            _lib.check(status, "PagedKVPool.decode_layers (peers)")
            return None
        status = lib.snapmind_paged_gqa_decode(
            q.data_ptr(), q.stride(1), q.stride(2), self.k.data_ptr(), self.v.data_ptr(), self._dcode,
            tables.data_ptr(), self.max_blocks_per_seq, self.max_blocks_per_seq, lens.data_ptr(),
            out.data_ptr(), out.stride(1), out.stride(2), float(scale), rows, n_q, self.n_kv_heads, self.head_dim,
            self.block_size, span, max_seq_len, split, 0, ws.data_ptr(), ws.numel(), self.err.data_ptr(),
            self._stream(),
        )  # fmt: skip
        _lib.check(status, "PagedKVPool.decode_layers")
        return out

    def decode(self, layer: int, q: torch.Tensor, out: torch.Tensor | None = None, scale: float | None = None,
               batch: int | None = None, split_tokens: int = 0, force_generic: bool = False,
               max_seq_len: int | None = None, peers=None, append=None, window: int = 0,
               sinks: int = 0, accumulate: bool = False) -> torch.Tensor | None:
        """Paged GQA decode attention of ``q`` ``[B, Hq, D]`` against layer ``layer``.

        With ``window`` > 0 a sequence attends to its last ``window`` tokens and its
        first ``sinks`` tokens only, and only their blocks are read (``split_tokens``
        and ``max_seq_len`` then have no use: the kernel plans from the device lengths).

        ``peers`` (a ``head_shard.PeerTargets``) sends the output rows to the
        output buffers of every rank of a head-sharded decode instead of ``out``
        and returns None.  ``append=(k_new, v_new)`` (``[B, H, D]``, the pool's
        dtype) stores this step's token of every sequence (the last slot the
        latest ``reserve(1)`` gave it) in the same launch, in place of an
        ``append`` call before the decode.  ``accumulate`` as in ``attend_chunk``."""
        if window or sinks or accumulate:
            if peers is not None:
                raise ValueError("decode with a window, or that accumulates, has no peer form")
            return self._attend_tokens(layer, q, out, scale, batch, window, sinks, force_generic, append, accumulate)
        batch = q.shape[0] if batch is None else batch
        n_q = q.shape[1]
        if peers is not None and append is not None:
            raise ValueError("decode with peers does not store the step's token: append it first")
        if q.dtype != self.dtype:
            raise TypeError(f"q dtype {q.dtype} != pool dtype {self.dtype}")
        if q.stride(-1) != 1:
            q = q.contiguous()
        if out is None and peers is None:
            out = torch.empty((batch, n_q, self.head_dim), dtype=self.dtype, device=self.device)
        scale = self.head_dim ** -0.5 if scale is None else scale
        if max_seq_len is None:
            max_seq_len = max(1, int(self._host_lens[:batch].max())) if batch else 1
        max_len = max_seq_len
        lib = _lib.load()
        split = split_tokens or lib.snapmind_paged_gqa_decode_split_tokens(
            batch, self.n_kv_heads, max_len, self.block_size
        )
        ws = self._decode_workspace(batch, n_q, max_len, split)
        if peers is not None:
            status = lib.snapmind_paged_gqa_decode_peers(
                q.data_ptr(), q.stride(0), q.stride(1),
                self.k[layer].data_ptr(), self.v[layer].data_ptr(), self._dcode,
                self.block_tables.data_ptr(), self.max_blocks_per_seq, self.max_blocks_per_seq,
                self.seq_lens.data_ptr(), None,
                peers.out_ptrs.data_ptr(), peers.n, peers.head_offset, peers.out_stride_seq, peers.out_stride_head,
                float(scale), batch, n_q, self.n_kv_heads, self.head_dim, self.block_size, self.num_blocks,
                max_len, split, _lib.DECODE_FORCE_GENERIC if force_generic else 0,
                ws.data_ptr(), ws.numel(), self.err.data_ptr(), self._stream(),
            )  # fmt: skip
            _lib.check(status, "PagedKVPool.decode (peers)")
            return None
        if append is not None:
            k_new, v_new = append
            if k_new.dtype != self.dtype or v_new.dtype != self.dtype or k_new.stride() != v_new.stride():
                raise TypeError("append rows must have the pool's dtype and matching strides")
            if k_new.shape != (batch, self.n_kv_heads, self.head_dim) or k_new.stride(-1) != 1:
                raise ValueError(f"append rows must be [{batch}, {self.n_kv_heads}, {self.head_dim}], "
                                 f"head dim contiguous, got {tuple(k_new.shape)}")
            status = lib.snapmind_paged_gqa_decode_append(
                q.data_ptr(), q.stride(0), q.stride(1),
                self.k[layer].data_ptr(), self.v[layer].data_ptr(), self._dcode,
                self.block_tables.data_ptr(), self.max_blocks_per_seq, self.max_blocks_per_seq,
                self.seq_lens.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), k_new.stride(0), k_new.stride(1),
                out.data_ptr(), out.stride(0), out.stride(1),
                float(scale), batch, n_q, self.n_kv_heads, self.head_dim, self.block_size, self.num_blocks,
                max_len, split, _lib.DECODE_FORCE_GENERIC if force_generic else 0,
                ws.data_ptr(), ws.numel(), self.err.data_ptr(), self._stream(),
            )  # fmt: skip
            _lib.check(status, "PagedKVPool.decode (append)")
            return out
        status = lib.snapmind_paged_gqa_decode(
            q.data_ptr(), q.stride(0), q.stride(1),
            self.k[layer].data_ptr(), self.v[layer].data_ptr(), self._dcode,
            self.block_tables.data_ptr(), self.max_blocks_per_seq, self.max_blocks_per_seq,
            self.seq_lens.data_ptr(),
            out.data_ptr(), out.stride(0), out.stride(1),
            float(scale), batch, n_q, self.n_kv_heads, self.head_dim, self.block_size, self.num_blocks,
            max_len, split, _lib.DECODE_FORCE_GENERIC if force_generic else 0,
            ws.data_ptr(), ws.numel(), self.err.data_ptr(), self._stream(),
        )  # fmt: skip
        _lib.check(status, "PagedKVPool.decode")
        return out

    def _lens_ladder(self, n: int) -> torch.Tensor:
        lad = getattr(self, "_ladder", None)
        if lad is None or lad.numel() < n:
            lad = torch.arange(1, max(n, 1) + 1, dtype=torch.int32, device=self.device)
            self._ladder = lad
        return lad

    def attend_causal(self, layer: int, b: int, q: torch.Tensor, out: torch.Tensor, n_b: int,
                      scale: float | None = None) -> torch.Tensor:
        """Causal attention of the newest ``T`` tokens of sequence ``b``
        (``q``/``out`` ``[Hq, T, D]``, sequence length ``n_b``): query t sees the
        first ``n_b - T + t + 1`` tokens; one decode-kernel row per query, all
        on the sequence's table row."""
        n_q, n_t = q.shape[0], q.shape[1]
        if n_t == 0:
            return out
        scale = self.head_dim ** -0.5 if scale is None else scale
        lad = self._lens_ladder(n_b)
        lib = _lib.load()
        split = lib.snapmind_paged_gqa_decode_split_tokens(n_t, self.n_kv_heads, n_b, self.block_size)
        ws = self._decode_workspace(n_t, n_q, n_b, split)
        status = lib.snapmind_paged_gqa_decode(
            q.data_ptr(), q.stride(1), q.stride(0),
            self.k[layer].data_ptr(), self.v[layer].data_ptr(), self._dcode,
            self.block_tables[b].data_ptr(), 0, self.max_blocks_per_seq, lad.data_ptr() + 4 * (n_b - n_t),
            out.data_ptr(), out.stride(1), out.stride(0),
            float(scale), n_t, n_q, self.n_kv_heads, self.head_dim, self.block_size, self.num_blocks,
            n_b, split, 0, ws.data_ptr(), ws.numel(), self.err.data_ptr(), self._stream(),
        )  # fmt: skip
        _lib.check(status, "PagedKVPool.attend_causal")
        return out

    def layer_views(self, batch: int) -> dict[int, "PoolLayerView"]:
        """One ``kv_cache`` view per layer for sequences ``0 .. batch - 1``."""
        return {i: PoolLayerView(self, i, batch) for i in range(self.n_layers)}


class PoolLayerView(MutableMapping):
    """The ``kv_cache`` of one layer for a batch of sequences of a
    :class:`PagedKVPool`, read and written by the ``gqa_paged`` attention plugin.

    The sequences are ragged, so the view holds no dense K/V tensor: ``"k"`` /
    ``"v"`` read as ``None`` until the layer has stored tokens (a model's prefill
    test, e.g. ``kv_cache.get("k") is None``) and as an empty placeholder after.
    The caller grows the sequences (``reserve``) before each forward; the
    plugin appends the new rows and attends from the pool.  ``capacity``, when
    set, is the length bound the decode split plan is made for (fixed plans
    for CUDA-graph replay).
    """

    KEYS = ("k", "v")

    def __init__(self, pool: PagedKVPool, layer: int, batch: int):
        self.pool, self.layer, self.batch = pool, layer, batch
        self.stored = 0
        self.capacity: int | None = None
        self._placeholder = torch.empty(0, dtype=pool.dtype, device=pool.device)

    def __getitem__(self, key):
        if key not in self.KEYS:
            raise KeyError(key)
        return None if self.stored == 0 else self._placeholder

    def __setitem__(self, key, value):
        raise TypeError("PoolLayerView is written by the gqa_paged attention plugin only")

    def __delitem__(self, key):
        raise TypeError("PoolLayerView entries cannot be deleted")

    def __iter__(self):
        return iter(self.KEYS)

    def __len__(self):
        return len(self.KEYS)
