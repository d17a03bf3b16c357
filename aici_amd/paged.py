"""Python handles on the C++ host side of the paged KV cache (csrc/hostkv.hip):
`BlockAllocator`, `BatchInfoBuilder`/`BatchInfo` and the cache geometry of
`CacheEngine` -- counterparts of rllm/rllm-cuda/src/llm/paged/*.rs.  All of it
runs on the host; torch is only used to hand the finished index arrays to the
GPU.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch

from . import _lib
from ._lib import call


class BlockAllocator:
    """blocks.rs:43-257."""

    def __init__(self, block_size: int, num_blocks: int):
        h = ctypes.c_void_p()
        call("hipattn_block_allocator_new", int(block_size), int(num_blocks), ctypes.byref(h))
        self._h = h
        self.block_size = int(block_size)
        self.num_blocks = int(num_blocks)

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h and _lib is not None:  # module globals are gone at interpreter shutdown
            _lib.load().hipattn_block_allocator_free(h)

    def get_num_free_blocks(self) -> int:
        return int(_lib.load().hipattn_block_allocator_num_free(self._h))

    def num_allocated_blocks(self, seq_id: int) -> int:
        return int(_lib.load().hipattn_block_allocator_num_allocated(self._h, int(seq_id)))

    def set_watermark(self, watermark: float) -> None:
        """blocks.rs:321-343: hold back `watermark * num_blocks` (truncated) blocks from new sequences."""
        call("hipattn_block_allocator_set_watermark", self._h, float(watermark))

    def can_allocate(self, seq_len: int) -> bool:
        """blocks.rs:267-270."""
        return bool(_lib.load().hipattn_block_allocator_can_allocate(self._h, int(seq_len)))

    def can_append_slot(self, num_running_seqs: int) -> bool:
        """blocks.rs:278-282."""
        return bool(_lib.load().hipattn_block_allocator_can_append_slot(self._h, int(num_running_seqs)))

    def alloc_seq(self, seq_id: int, seq_len: int) -> None:
        call("hipattn_block_allocator_alloc_seq", self._h, int(seq_id), int(seq_len))

    def append_slots(self, seq_id: int, num_kv_computed: int, seq_len: int) -> List[Tuple[int, int]]:
        """Returns the (old, new) block pairs the caller must copy (copy-on-write)."""
        cap = (int(seq_len) + self.block_size - 1) // self.block_size + 1
        buf = (ctypes.c_int64 * (2 * cap))()
        n = ctypes.c_int64()
        call("hipattn_block_allocator_append_slots", self._h, int(seq_id), int(num_kv_computed), int(seq_len), buf,
             cap, ctypes.byref(n))
        return [(int(buf[2 * i]), int(buf[2 * i + 1])) for i in range(n.value)]

    def step_generation(self, seq_ids: Sequence[int], seq_lens: Sequence[int], num_kv_computed: Sequence[int]):
        """scheduler.rs:304-337 + 357-380 for groups of one sequence (ids in arrival order): returns
        (scheduled ids, preempted ids, copy-on-write pairs).  A preempted sequence holds no blocks any more
        and has to be admitted and recomputed."""
        n = len(seq_ids)
        ids = (ctypes.c_int64 * max(1, n))(*[int(x) for x in seq_ids])
        lens = (ctypes.c_int64 * max(1, n))(*[int(x) for x in seq_lens])
        comp = (ctypes.c_int64 * max(1, n))(*[int(x) for x in num_kv_computed])
        sched, pre = (ctypes.c_int64 * max(1, n))(), (ctypes.c_int64 * max(1, n))()
        cap = sum((int(l) + self.block_size - 1) // self.block_size + 1 for l in seq_lens) + 1
        pairs = (ctypes.c_int64 * (2 * cap))()
        ns, np_, npairs = ctypes.c_int64(), ctypes.c_int64(), ctypes.c_int64()
        call("hipattn_block_allocator_step_generation", self._h, ids, lens, comp, n, sched, ctypes.byref(ns), pre,
             ctypes.byref(np_), pairs, cap, ctypes.byref(npairs))
        return ([int(sched[i]) for i in range(ns.value)], [int(pre[i]) for i in range(np_.value)],
                [(int(pairs[2 * i]), int(pairs[2 * i + 1])) for i in range(npairs.value)])

    def copy(self, src: int, dst: int, length: int) -> None:
        call("hipattn_block_allocator_copy", self._h, int(src), int(dst), int(length))

    def trim(self, seq_id: int, length: int) -> None:
        call("hipattn_block_allocator_trim", self._h, int(seq_id), int(length))

    def delete(self, seq_id: int) -> None:
        call("hipattn_block_allocator_delete", self._h, int(seq_id))

    def get_block_idxes(self, seq_id: int, length: int) -> np.ndarray:
        out = np.empty((int(length),), dtype=np.int64)
        call("hipattn_block_allocator_get_block_idxes", self._h, int(seq_id), int(length),
             out.ctypes.data_as(ctypes.POINTER(ctypes.c_int64)))
        return out

    def swap_out(self, seq_id: int) -> List[int]:
        """blocks.rs:176-189: the sequence's blocks (logical order), released here."""
        n = ctypes.c_int64()
        call("hipattn_block_allocator_swap_out", self._h, int(seq_id), None, 0, ctypes.byref(n))
        buf = (ctypes.c_int64 * max(1, n.value))()
        call("hipattn_block_allocator_swap_out", self._h, int(seq_id), buf, n.value, ctypes.byref(n))
        return [int(buf[i]) for i in range(n.value)]

    def swap_in(self, seq_id: int, block_idxs: Sequence[int], mapping: dict) -> None:
        """blocks.rs:191-210: one block here per entry of block_idxs (blocks of the other allocator);
        `mapping` (other-side block -> block here) is shared by the sequences of a group and extended."""
        n = len(block_idxs)
        src = (ctypes.c_int64 * max(1, n))(*[int(b) for b in block_idxs])
        cap = len(mapping) + n
        pairs = (ctypes.c_int64 * max(1, 2 * cap))()
        for i, (k, v) in enumerate(mapping.items()):
            pairs[2 * i], pairs[2 * i + 1] = int(k), int(v)
        used = ctypes.c_int64(len(mapping))
        call("hipattn_block_allocator_swap_in", self._h, int(seq_id), src, n, pairs, cap, ctypes.byref(used))
        for i in range(len(mapping), used.value):
            mapping[int(pairs[2 * i])] = int(pairs[2 * i + 1])


# SchedulingPhase (seq.rs:44-51) and what `BlockSpaceManager.step_generation` did with a group.
SEQ_RUNNING, SEQ_SUSPENDED, SEQ_SWAPPED, SEQ_WAITING, SEQ_FINISHED = range(5)
GROUP_NOT_REACHED, GROUP_SCHEDULED, GROUP_SUSPENDED, GROUP_RECOMPUTE, GROUP_SWAPPED_OUT = -1, 0, 1, 2, 3


class BlockSpaceManager:
    """blocks.rs:259-380: the mapping between logical and physical blocks on both sides of the swap --
    a device allocator with its admission watermark and a host allocator.  Sequences are plain ids;
    a group is a list of ids (the reference's SequenceGroup carries the scheduling phase itself, here
    the caller says which of the group's sequences are running or swapped)."""

    def __init__(self, block_size: int, num_gpu_blocks: int, num_cpu_blocks: int, watermark: float = 0.01):
        assert watermark >= 0.0
        self.gpu_allocator = BlockAllocator(block_size, num_gpu_blocks)
        self.cpu_allocator = BlockAllocator(block_size, num_cpu_blocks)
        self.gpu_allocator.set_watermark(watermark)
        self.watermark_blocks = int(watermark * num_gpu_blocks)

    def can_allocate(self, seq_len: int) -> bool:
        return self.gpu_allocator.can_allocate(seq_len)                                   # :266-270

    def allocate(self, seq_id: int, seq_len: int) -> None:
        self.gpu_allocator.alloc_seq(seq_id, seq_len)                                     # :272-276

    def can_append_slot(self, num_running_seqs: int) -> bool:
        return self.gpu_allocator.can_append_slot(num_running_seqs)                       # :278-282

    def append_slots(self, seq_id: int, num_kv_computed: int, seq_len: int) -> List[Tuple[int, int]]:
        return self.gpu_allocator.append_slots(seq_id, num_kv_computed, seq_len)          # :284-286

    def num_phys_blocks(self, seq_ids: Sequence[int]) -> int:
        total = 0                                                                         # :364-379
        for s in seq_ids:
            n = self.gpu_allocator.num_allocated_blocks(s)
            if n == 0:
                n = self.cpu_allocator.num_allocated_blocks(s)
            else:
                assert self.cpu_allocator.num_allocated_blocks(s) == 0
            total += n
        return total

    def can_swap_in(self, seq_ids: Sequence[int], num_swapped_seqs: Optional[int] = None) -> bool:
        n = len(seq_ids) if num_swapped_seqs is None else num_swapped_seqs               # :288-293
        need = self.num_phys_blocks(seq_ids) + n + self.watermark_blocks
        return self.gpu_allocator.get_num_free_blocks() >= need

    def swap_in(self, swapped_seq_ids: Sequence[int]) -> dict:
        """:295-305.  Returns host block -> device block for `CacheEngine.swap_in`."""
        mapping: dict = {}
        for s in swapped_seq_ids:
            self.gpu_allocator.swap_in(s, self.cpu_allocator.swap_out(s), mapping)
        return mapping

    def can_swap_out(self, seq_ids: Sequence[int]) -> bool:
        return self.num_phys_blocks(seq_ids) <= self.cpu_allocator.get_num_free_blocks()  # :319-322

    def swap_out(self, running_seq_ids: Sequence[int]) -> dict:
        """:307-317.  Returns device block -> host block for `CacheEngine.swap_out`."""
        mapping: dict = {}
        for s in running_seq_ids:
            self.cpu_allocator.swap_in(s, self.gpu_allocator.swap_out(s), mapping)
        return mapping

    def step_generation(self, groups: Sequence[Tuple[int, Sequence[Tuple[int, int, int, int]]]]) -> dict:
        """scheduler.rs:304-337, 346-380 for sequence groups of any size.  groups, in arrival order, are
        (max_running_seqs, [(seq_id, phase, seq_len to grow to, num_kv_computed), ...]) with phase one of
        SEQ_RUNNING .. SEQ_FINISHED.  Returns {"fates": one GROUP_* per group, "copies": copy-on-write
        (old, new) device block pairs, "swap_out": (device block, host block) pairs for
        `CacheEngine.swap_out`}."""
        starts, ids, phases, lens, comp, maxrun = [0], [], [], [], [], []
        for max_running, seqs in groups:
            maxrun.append(int(max_running))
            for sid, phase, seq_len, computed in seqs:
                ids.append(int(sid))
                phases.append(int(phase))
                lens.append(int(seq_len))
                comp.append(int(computed))
            starts.append(len(ids))
        g, n = len(maxrun), len(ids)
        bs = self.gpu_allocator.block_size
        cap_copy = sum((l + bs - 1) // bs + 1 for l in lens) + 1
        cap_swap = sum(self.gpu_allocator.num_allocated_blocks(s) for s in ids) + 1
        a64 = lambda v: (ctypes.c_int64 * max(1, len(v)))(*v)
        fates = (ctypes.c_int32 * max(1, g))()
        copies, swaps = (ctypes.c_int64 * (2 * cap_copy))(), (ctypes.c_int64 * (2 * cap_swap))()
        nc, nsw = ctypes.c_int64(), ctypes.c_int64()
        call("hipattn_block_space_step_generation", self.gpu_allocator._h, self.cpu_allocator._h, g, a64(starts),
             a64(maxrun), a64(ids), (ctypes.c_int32 * max(1, n))(*phases), a64(lens), a64(comp), fates, copies,
             cap_copy, ctypes.byref(nc), swaps, cap_swap, ctypes.byref(nsw))
        return {"fates": [int(fates[i]) for i in range(g)],
                "copies": [(int(copies[2 * i]), int(copies[2 * i + 1])) for i in range(nc.value)],
                "swap_out": [(int(swaps[2 * i]), int(swaps[2 * i + 1])) for i in range(nsw.value)]}

    def get_num_free_gpu_blocks(self) -> int:
        return self.gpu_allocator.get_num_free_blocks()

    def get_num_free_cpu_blocks(self) -> int:
        return self.cpu_allocator.get_num_free_blocks()

    # TchSeqMgr (blocks.rs:382-443): fork / trim / delete act on both sides
    def copy(self, src: int, dst: int, length: int) -> None:
        self.cpu_allocator.copy(src, dst, length)
        self.gpu_allocator.copy(src, dst, length)

    def trim(self, seq_id: int, length: int) -> None:
        self.cpu_allocator.trim(seq_id, length)
        self.gpu_allocator.trim(seq_id, length)

    def delete(self, seq_id: int) -> None:
        self.cpu_allocator.delete(seq_id)
        self.gpu_allocator.delete(seq_id)


@dataclass
class BatchInfo:
    """batch_info.rs:18-43 (host copies; `to(device)` uploads what the kernels read)."""
    tokens: torch.Tensor
    positions: torch.Tensor
    seqlens_q: torch.Tensor
    seqlens_k: torch.Tensor
    gather_mapping: torch.Tensor
    slot_mapping: torch.Tensor
    logit_idxs: torch.Tensor
    max_seqlen_q: int
    max_seqlen_k: int
    seq_ids: List[int]
    paged_block_tables: torch.Tensor
    paged_context_lens: torch.Tensor
    paged_block_size: int
    paged_max_context_len: int
    seqlen_multi: int
    q_multi: int
    # extension: block tables / key counts of the multi-token entries (None when some entry's slots do not
    # walk its blocks in order, in which case only the gather route applies)
    multi_block_tables: Optional[torch.Tensor] = None
    multi_context_lens: Optional[torch.Tensor] = None

    def to(self, device) -> "BatchInfo":
        """The batch with its arrays on `device`, there when the call returns: they may be used on any stream.  On the way
        from the host to a GPU all of them travel as one copy, waited for once: a pageable copy per array costs some
        12 us, the wait included, and a step has ten of them."""
        device = torch.device(device)
        tensors = {k: v for k, v in self.__dict__.items() if isinstance(v, torch.Tensor)}
        kw = dict(self.__dict__)
        if device.type != "cuda" or not all(v.device.type == "cpu" and v.is_contiguous() and v.dtype in (torch.int32, torch.int64)
                                            for v in tensors.values()):
            kw.update((k, v.to(device)) for k, v in tensors.items())
            return BatchInfo(**kw)
        # in words of 4 bytes, every array on a 16-byte boundary
        words = [v.numel() * v.element_size() // 4 for v in tensors.values()]
        padded = [(w + 3) & ~3 for w in words]
        staged = torch.empty((sum(padded),), dtype=torch.int32, pin_memory=True)
        host, at = staged.numpy(), 0
        for v, w, p in zip(tensors.values(), words, padded):
            if w:
                host[at:at + w] = v.numpy().reshape(-1).view(np.int32)
            at += p
        there = torch.empty((sum(padded),), dtype=torch.int32, device=device)
        for (k, v), w, part in zip(tensors.items(), words, there.split(padded)):
            if w != part.numel():
                part = part[:w]
            kw[k] = (part if v.dtype == torch.int32 else part.view(v.dtype)).view(v.shape)
        batch = BatchInfo(**kw)
        there.copy_(staged)  # waits for the copy, and so for the work queued before it: nothing is left to do behind it
        return batch


def _np(ptr, n: int, dtype) -> np.ndarray:
    if n == 0:
        return np.zeros((0,), dtype=dtype)
    return np.ctypeslib.as_array(ptr, shape=(n,)).astype(dtype, copy=True)


class BatchInfoBuilder:
    """batch_info.rs:103-315."""

    def __init__(self, block_size: int, max_model_len: int, paged_attn_kernel_v: int = 1):
        h = ctypes.c_void_p()
        call("hipattn_batch_builder_new", int(block_size), int(max_model_len), int(paged_attn_kernel_v),
             ctypes.byref(h))
        self._h = h

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h and _lib is not None:
            _lib.load().hipattn_batch_builder_free(h)

    def add_entry(self, seq_id: int, query_positions: Sequence[int], query_tokens: Sequence[int],
                  kv_slots: Sequence[int]) -> "BatchInfoBuilder":
        qp = np.ascontiguousarray(query_positions, dtype=np.int64)
        qt = np.ascontiguousarray(query_tokens, dtype=np.int32)
        ks = np.ascontiguousarray(kv_slots, dtype=np.int64)
        call("hipattn_batch_builder_add", self._h, int(seq_id), qp.ctypes.data_as(ctypes.POINTER(ctypes.c_int64)),
             qt.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)), len(qp),
             ks.ctypes.data_as(ctypes.POINTER(ctypes.c_int64)), len(ks))
        return self

    def sched_out(self, alloc: BlockAllocator, seq_id: int, seq_tokens: Sequence[int],
                  num_kv_computed: int) -> "BatchInfoBuilder":
        st = np.ascontiguousarray(seq_tokens, dtype=np.int32)
        call("hipattn_batch_builder_add_seq", self._h, alloc._h, int(seq_id),
             st.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)), len(st), int(num_kv_computed))
        return self

    def finish(self) -> BatchInfo:
        bi = _lib.BatchInfo()
        call("hipattn_batch_builder_finish", self._h, ctypes.byref(bi))
        return _batch_info(bi)


class DecodeBatch:
    """The single-token rows of a running batch kept across steps (`hipattn_decode_batch`): `info()` equals
    what `BatchInfoBuilder.finish()` gives for the same sequences in the same order, without the per-step
    rebuild from every sequence's full slot list (batch_info.rs:196-315)."""

    def __init__(self, block_size: int, max_model_len: int):
        h = ctypes.c_void_p()
        call("hipattn_decode_batch_new", int(block_size), int(max_model_len), ctypes.byref(h))
        self._h = h

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h and _lib is not None:
            _lib.load().hipattn_decode_batch_free(h)

    def __len__(self) -> int:
        return int(_lib.load().hipattn_decode_batch_size(self._h))

    def add(self, alloc: BlockAllocator, seq_id: int, last_token: int, seq_len: int) -> None:
        call("hipattn_decode_batch_add", self._h, alloc._h, int(seq_id), int(last_token), int(seq_len))

    def advance(self, alloc: BlockAllocator, seq_id: int, new_token: int) -> None:
        call("hipattn_decode_batch_advance", self._h, alloc._h, int(seq_id), int(new_token))

    def advance_all(self, alloc: BlockAllocator, new_tokens: Sequence[int]) -> None:
        """One generation step for every row: new_tokens[i] is row i's new token."""
        t = np.ascontiguousarray(new_tokens, dtype=np.int32)
        call("hipattn_decode_batch_advance_all", self._h, alloc._h, t.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)),
             len(t))

    def remove(self, seq_id: int) -> None:
        call("hipattn_decode_batch_remove", self._h, int(seq_id))

    def info(self) -> BatchInfo:
        bi = _lib.BatchInfo()
        call("hipattn_decode_batch_info", self._h, ctypes.byref(bi))
        return _batch_info(bi)


class DeviceBlocks:
    """The blocks of a paged cache on the device (`kernels.step_blocks`), for up to max_requests requests that share none: every step's block
    tables, slots and positions come from how many tokens each request brings, without the host knowing a length, so that a step can be
    captured into a graph.  With a window (window_size_left >= 0, as in `attn.varlen_attn`) blocks that it has passed, sinks aside,
    go back to the pool: the window of every layer, as the layers share the tables.  A request is a row of the tables; the row is free again
    when its request has ended."""

    def __init__(self, block_size: int, num_blocks: int, max_requests: int, max_model_len: int, device, window_size_left: int = -1,
                 sink_tokens: int = 0):
        self.block_size = int(block_size)
        self.window_size_left, self.sink_tokens = int(window_size_left), int(sink_tokens)
        columns = (int(max_model_len) + self.block_size - 1) // self.block_size
        self.max_context_len = columns * self.block_size
        self.state = torch.zeros((max_requests, 2), dtype=torch.int32, device=device)
        self.block_tables = torch.zeros((max_requests, columns), dtype=torch.int32, device=device)
        self.free_ring = torch.arange(num_blocks, dtype=torch.int32, device=device)
        self.ring_ends = torch.tensor([0, num_blocks], dtype=torch.int64, device=device)

    def step(self, new_lens: torch.Tensor, num_rows: int, rows_per_request: int = 0):
        """int32 [max_requests] tokens that every request brings (0: idle, negative: ended) -> `kernels.StepBlocks` of num_rows rows."""
        from . import kernels

        return kernels.step_blocks(new_lens, self.state, self.block_tables, self.free_ring, self.ring_ends, self.block_size, num_rows,
                                   rows_per_request, self.window_size_left, self.sink_tokens, state_out=self.state,
                                   ring_ends_out=self.ring_ends)

    def batch_info(self, step, tokens: torch.Tensor, max_new: Optional[int] = None) -> BatchInfo:
        """The batch of a step whose rows hold `tokens` [num_rows].  max_new None: decode rows, of a step with rows_per_request=1 and a row for
        every request; else chunks of at most max_new tokens, of a step with rows_per_request=0, read through the block tables."""
        rows, requests = step.positions.numel(), self.state.size(0)
        decode = max_new is None
        if decode and rows != requests:
            raise ValueError(f"decode rows: {rows} rows for {requests} requests")
        none = self.free_ring.new_zeros((0,))
        return BatchInfo(
            tokens=tokens, positions=step.positions, seqlens_q=none if decode else step.seqlens_q, seqlens_k=none, gather_mapping=none,
            slot_mapping=step.slot_mapping, logit_idxs=step.logit_idxs, max_seqlen_q=0 if decode else int(max_new),
            max_seqlen_k=0 if decode else self.max_context_len, seq_ids=list(range(requests)),
            paged_block_tables=self.block_tables if decode else none.view(0, 0),
            paged_context_lens=step.context_lens if decode else none, paged_block_size=self.block_size,
            paged_max_context_len=self.max_context_len if decode else 0, seqlen_multi=0 if decode else requests,
            q_multi=0 if decode else rows, multi_block_tables=None if decode else self.block_tables,
            multi_context_lens=None if decode else step.context_lens)


def _batch_info(bi) -> BatchInfo:
    """Copies a `hipattn_batch_info` (arrays owned by the C++ side) into host tensors."""
    nm = int(bi.num_multi)
    tables = _np(bi.paged_block_tables, int(bi.num_paged * bi.paged_max_blocks), np.int32)
    return BatchInfo(
        tokens=torch.from_numpy(_np(bi.tokens, int(bi.num_tokens), np.int32)),
        positions=torch.from_numpy(_np(bi.positions, int(bi.num_tokens), np.int64)),
        seqlens_q=torch.from_numpy(_np(bi.seqlens_q, nm + 1, np.int32)),
        seqlens_k=torch.from_numpy(_np(bi.seqlens_k, nm + 1, np.int32)),
        gather_mapping=torch.from_numpy(_np(bi.gather_mapping, int(bi.num_gather), np.int32)),
        slot_mapping=torch.from_numpy(_np(bi.slot_mapping, int(bi.num_tokens), np.int32)),
        logit_idxs=torch.from_numpy(_np(bi.logit_idxs, int(bi.num_seqs), np.int32)),
        max_seqlen_q=int(bi.max_seqlen_q),
        max_seqlen_k=int(bi.max_seqlen_k),
        seq_ids=[int(x) for x in _np(bi.seq_ids, int(bi.num_seqs), np.int64)],
        paged_block_tables=torch.from_numpy(tables).reshape(int(bi.num_paged), int(bi.paged_max_blocks)),
        paged_context_lens=torch.from_numpy(_np(bi.paged_context_lens, int(bi.num_paged), np.int32)),
        paged_block_size=int(bi.paged_block_size),
        paged_max_context_len=int(bi.paged_max_context_len),
        seqlen_multi=nm,
        q_multi=int(bi.q_multi),
        multi_block_tables=(torch.from_numpy(_np(bi.multi_block_tables, nm * int(bi.multi_max_blocks), np.int32))
                            .reshape(nm, int(bi.multi_max_blocks)) if bi.multi_tables_valid else None),
        multi_context_lens=(torch.from_numpy(_np(bi.multi_context_lens, nm, np.int32))
                            if bi.multi_tables_valid else None),
    )


_DT = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def cache_x(dtype: torch.dtype) -> int:
    """cache_engine.rs:85: elements per 16-byte run of the key cache."""
    return int(_lib.load().hipattn_cache_x(_DT[dtype]))


def cache_block_bytes(block_size: int, num_kv_heads: int, head_size: int, num_layers: int,
                      dtype: torch.dtype) -> int:
    """cache_engine.rs:165-175 `get_cache_block_size`."""
    return int(_lib.load().hipattn_cache_block_bytes(block_size, num_kv_heads, head_size, num_layers, _DT[dtype]))


def alloc_gpu_cache_layer(num_blocks: int, num_kv_heads: int, head_size: int, block_size: int, dtype: torch.dtype,
                          device) -> Tuple[torch.Tensor, torch.Tensor]:
    """cache_engine.rs:81-111: K [nb,Hkv,d/x,BS,x] and V [nb,Hkv,d,BS], uninitialised."""
    x = cache_x(dtype)
    k = torch.empty((num_blocks, num_kv_heads, head_size // x, block_size, x), dtype=dtype, device=device)
    v = torch.empty((num_blocks, num_kv_heads, head_size, block_size), dtype=dtype, device=device)
    return k, v


class CacheEngine:
    """cache_engine.rs:16-176: the per-layer paged K/V caches on the device, their host-side swap
    space, the side stream that block swaps run on with one event per layer, and copy-on-write
    block copies.  Host caches are pinned (allocated so, never registered afterwards)."""

    def __init__(self, num_layers: int, num_kv_heads: int, head_size: int, block_size: int, dtype: torch.dtype,
                 num_gpu_blocks: int, num_cpu_blocks: int, device):
        from . import kernels

        self._k = kernels
        self.device = torch.device(device)
        self.block_size = block_size
        self.gpu_cache = [alloc_gpu_cache_layer(num_gpu_blocks, num_kv_heads, head_size, block_size, dtype, self.device)
                          for _ in range(num_layers)]                                      # :117-121
        x = cache_x(dtype)
        self.cpu_cache = [(torch.empty((num_cpu_blocks, num_kv_heads, head_size // x, block_size, x), dtype=dtype,
                                       pin_memory=num_cpu_blocks > 0),
                           torch.empty((num_cpu_blocks, num_kv_heads, head_size, block_size), dtype=dtype,
                                       pin_memory=num_cpu_blocks > 0)) for _ in range(num_layers)]  # :123-133
        index = self.device.index or 0
        self.cache_stream = kernels.CudaStream(kernels.CudaStream.LOW_PRI, index)          # :47
        self.events = [kernels.CudaEvent() for _ in range(num_layers)]                     # :48
        self.used_events = False

    def get_cache_iface(self):
        """:53-66.  Returns get(layer) -> (key_cache, value_cache); when a swap was issued this round the
        calling thread's current stream first waits for that layer's swap to land."""
        events = self.events if self.used_events else None
        stream = self._k.CudaStream.current(self.device.index or 0)
        gpu_cache = self.gpu_cache

        def get(layer_no: int) -> Tuple[torch.Tensor, torch.Tensor]:
            if events is not None:
                events[layer_no].wait(stream)
            return gpu_cache[layer_no]

        return get

    def new_round(self) -> None:
        self.used_events = False                                                           # :68-70

    def swap_in(self, src_to_dst) -> None:
        self._swap(self.cpu_cache, self.gpu_cache, src_to_dst)                             # :72-75
        self.used_events = True

    def swap_out(self, src_to_dst) -> None:
        self._swap(self.gpu_cache, self.cpu_cache, src_to_dst)                             # :77-80
        self.used_events = True

    def _swap(self, src, dst, src_to_dst) -> None:
        """:145-155: every layer's K then V on the cache stream, the layer's event recorded after them."""
        for i, (src_k, src_v) in enumerate(src):
            dst_k, dst_v = dst[i]
            self._k.swap_blocks(src_k, dst_k, src_to_dst, self.cache_stream)
            self._k.swap_blocks(src_v, dst_v, src_to_dst, self.cache_stream)
            self.events[i].record(self.cache_stream)

    def copy(self, src_to_dsts) -> None:
        """:157-169: copy-on-write copies in all layers at once."""
        self._k.copy_blocks([k for k, _ in self.gpu_cache], [v for _, v in self.gpu_cache], src_to_dsts)

    @staticmethod
    def get_cache_block_size(block_size: int, num_kv_heads: int, head_size: int, num_layers: int,
                             dtype: torch.dtype) -> int:
        return cache_block_bytes(block_size, num_kv_heads, head_size, num_layers, dtype)   # :171-175
