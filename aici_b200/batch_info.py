"""Host-side mirror of rLLM's BatchInfoBuilder / BatchInfo for the attention path.

Same roles and field names as rllm-cuda/src/llm/paged/batch_info.rs (BatchEntry :93-97,
BatchInfoBuilder :88-315, BatchInfo :18-43).  The work is done by the native builder behind
`aici_batch_info_build` (include/aici_b200.h): every index tensor of the step is written into one
page-locked staging buffer and reaches the device with one copy; the fields of the returned
`BatchInfo` are views into that one device buffer.
"""
import ctypes
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import _lib
from ._lib import AiciError
from .tch_cuda import _call, _one_gpu

PAGED_DECODE = 1
TABLES_FOR_ALL = 2
NO_GATHER_MAP = 4


class _Entry(ctypes.Structure):
    _fields_ = [("seq_id", ctypes.c_int64), ("tokens", ctypes.c_void_p),
                ("positions", ctypes.c_void_p), ("kv_slots", ctypes.c_void_p),
                ("q_len", ctypes.c_int32), ("k_len", ctypes.c_int32)]


class Layout(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in (
        "total_bytes", "tokens_off", "positions_off", "slot_mapping_off", "logit_idxs_off",
        "seqlens_q_off", "seqlens_k_off", "gather_mapping_off", "block_tables_off",
        "context_lens_off")] + [(n, ctypes.c_int32) for n in (
            "num_entries", "num_tokens", "num_multitoken", "q_multi", "max_seqlen_q", "max_seqlen_k",
            "gather_len", "num_paged", "table_rows", "paged_row0", "max_blocks_per_seq",
            "paged_max_context_len")]


class BatchInfo:
    """Index tensors of one step (batch_info.rs:18-43); all views of `buffer`."""

    def __init__(self, buffer: torch.Tensor, lay: Layout, order: List[int], seq_ids: List[int],
                 block_size: int, step_no: int):
        def sec(off, count, dtype):
            nbytes = count * torch.empty((), dtype=dtype).element_size()
            return buffer[off:off + nbytes].view(dtype)

        self.buffer = buffer
        self.layout = lay
        self.step_no = step_no
        self.tokens = sec(lay.tokens_off, lay.num_tokens, torch.int32)
        self.positions = sec(lay.positions_off, lay.num_tokens, torch.int64)
        self.slot_mapping = sec(lay.slot_mapping_off, lay.num_tokens, torch.int32)
        self.logit_idxs = sec(lay.logit_idxs_off, lay.num_entries, torch.int32)
        self.seqlens_q = sec(lay.seqlens_q_off, lay.num_multitoken + 1, torch.int32)
        self.seqlens_k = sec(lay.seqlens_k_off, lay.num_multitoken + 1, torch.int32)
        self.gather_mapping = sec(lay.gather_mapping_off, lay.gather_len, torch.int32)
        tables = sec(lay.block_tables_off, lay.table_rows * lay.max_blocks_per_seq, torch.int32)
        tables = tables.view(lay.table_rows, lay.max_blocks_per_seq)
        lens = sec(lay.context_lens_off, lay.table_rows, torch.int32)
        # rows of the single-token entries, as the reference's fields of the same name
        self.paged_block_tables = tables[lay.paged_row0:]
        self.paged_context_lens = lens[lay.paged_row0:]
        # rows of the multi-token entries (empty unless TABLES_FOR_ALL was asked for)
        self.multi_block_tables = tables[:lay.paged_row0]
        self.multi_context_lens = lens[:lay.paged_row0]
        self.paged_block_size = block_size
        self.paged_max_context_len = lay.paged_max_context_len
        self.max_seqlen_q = lay.max_seqlen_q
        self.max_seqlen_k = lay.max_seqlen_k
        self.seqlen_multi = lay.num_multitoken
        self.q_multi = lay.q_multi
        self.entry_order = order
        self.seq_id_to_idx: Dict[int, int] = {seq_ids[e]: i for i, e in enumerate(order)}


class BatchInfoBuilder:
    """Collects the running sequences of a step, then `finish()` lays them out and uploads them.

    `paged_attn_kernel_v`, `block_size`, `max_model_len` are the config fields the reference
    reads (batch_info.rs:209, 223, 249).  The staging buffers (host, page-locked when a device
    is given) are kept and grown between steps, so a steady-state step allocates nothing.
    """

    def __init__(self, block_size: int = 16, max_model_len: int = 1 << 20,
                 paged_attn_kernel_v: int = 1, device: Optional[torch.device] = None,
                 tables_for_all: bool = False, gather_mapping: bool = True):
        self.block_size = block_size
        self.max_model_len = max_model_len
        self.flags = ((PAGED_DECODE if paged_attn_kernel_v > 0 else 0) |
                      (TABLES_FOR_ALL if tables_for_all else 0) |
                      (0 if gather_mapping else NO_GATHER_MAP))
        self.device = device
        self.entries: List[Tuple[int, torch.Tensor, Optional[torch.Tensor], torch.Tensor]] = []
        # two staging buffers used in turn; each remembers the event of its last upload
        self._staging: List[Optional[torch.Tensor]] = [None, None]
        self._uploaded: List[Optional[torch.cuda.Event]] = [None, None]
        self._turn = 0

    def add_entry(self, seq_id: int, query_pos_token: Sequence[Tuple[int, int]],
                  kv_slots: Sequence[int]) -> "BatchInfoBuilder":
        """One BatchEntry (batch_info.rs:93-97): (position, token) pairs of this step's query
        tokens and the cache slot of every token of the sequence."""
        pos = torch.tensor([p for p, _ in query_pos_token], dtype=torch.int64)
        tok = torch.tensor([t for _, t in query_pos_token], dtype=torch.int32)
        slots = torch.as_tensor(kv_slots, dtype=torch.int64).contiguous()
        self.entries.append((int(seq_id), tok, pos, slots))
        return self

    def add_arrays(self, seq_id: int, tokens: torch.Tensor, kv_slots: torch.Tensor,
                   positions: Optional[torch.Tensor] = None) -> "BatchInfoBuilder":
        """Same entry from ready-made CPU arrays (int32 tokens, int64 slots); positions default to
        the last len(tokens) positions of the sequence, which is what sched_out produces
        (batch_info.rs:121-140)."""
        self.entries.append((int(seq_id), tokens.to(torch.int32).contiguous(),
                             None if positions is None else positions.to(torch.int64).contiguous(),
                             kv_slots.to(torch.int64).contiguous()))
        return self

    def _c_entries(self):
        arr = (_Entry * max(len(self.entries), 1))()
        for i, (seq_id, tok, pos, slots) in enumerate(self.entries):
            arr[i].seq_id = seq_id
            arr[i].tokens = tok.data_ptr()
            arr[i].positions = 0 if pos is None else pos.data_ptr()
            arr[i].kv_slots = slots.data_ptr()
            arr[i].q_len = tok.numel()
            arr[i].k_len = slots.numel()
        return arr

    def finish(self, step_no: int = 0) -> BatchInfo:
        """BatchInfoBuilder::finish (batch_info.rs:196-315).  Clears the entry list."""
        fn = "BatchInfoBuilder.finish"
        n = len(self.entries)
        arr = self._c_entries()
        lay = Layout()
        lib = _lib.lib()
        _lib.check(fn, lib.aici_batch_info_layout(arr, ctypes.c_int(n), ctypes.c_int(self.flags),
                                                  ctypes.c_int(self.block_size),
                                                  ctypes.c_int64(self.max_model_len), ctypes.byref(lay)))
        need = max(int(lay.total_bytes), 256)
        on_gpu = self.device is not None and torch.device(self.device).type == "cuda"
        turn = self._turn
        self._turn ^= 1
        if self._staging[turn] is None or self._staging[turn].numel() < need:
            self._staging[turn] = torch.empty(max(need * 2, 1 << 16), dtype=torch.uint8,
                                              pin_memory=on_gpu)
        elif self._uploaded[turn] is not None:
            self._uploaded[turn].synchronize()  # the copy that last read this buffer is done
        staging = self._staging[turn]
        order = (ctypes.c_int32 * n)()
        if on_gpu:
            dev = torch.device(self.device)
            with torch.cuda.device(dev):
                buffer = torch.empty(need, dtype=torch.uint8, device=dev)
                _lib.check(fn, lib.aici_batch_info_build(
                    arr, ctypes.c_int(n), ctypes.c_int(self.flags), ctypes.c_int(self.block_size),
                    ctypes.c_int64(self.max_model_len), ctypes.c_void_p(staging.data_ptr()),
                    ctypes.c_size_t(staging.numel()), ctypes.c_void_p(buffer.data_ptr()),
                    ctypes.c_size_t(buffer.numel()), ctypes.byref(lay), order,
                    ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)))
                ev = torch.cuda.Event()
                ev.record()
                self._uploaded[turn] = ev
        else:
            _lib.check(fn, lib.aici_batch_info_build(
                arr, ctypes.c_int(n), ctypes.c_int(self.flags), ctypes.c_int(self.block_size),
                ctypes.c_int64(self.max_model_len), ctypes.c_void_p(staging.data_ptr()),
                ctypes.c_size_t(staging.numel()), ctypes.c_void_p(0), ctypes.c_size_t(0),
                ctypes.byref(lay), order, ctypes.c_void_p(0)))
            buffer = staging[:need].clone()
        seq_ids = [e[0] for e in self.entries]
        self.entries = []
        return BatchInfo(buffer, lay, list(order), seq_ids, self.block_size, step_no)


class StepTables:
    """Index tensors of one step, built on the GPU by `step_tables` (fields as in BatchInfo)."""
    __slots__ = ("seqlens_q", "positions", "slot_mapping", "logit_idxs", "context_lens", "free_count")

    def __init__(self, seqlens_q, positions, slot_mapping, logit_idxs, context_lens, free_count):
        self.seqlens_q = seqlens_q        # int32 [requests + 1]
        self.positions = positions        # int64 [max_tokens], 0 behind the last token
        self.slot_mapping = slot_mapping  # int32 [max_tokens], -1 behind the last token
        self.logit_idxs = logit_idxs      # int32 [requests], -1 for a request without new tokens
        self.context_lens = context_lens  # int32 [requests], new tokens included
        self.free_count = free_count      # int32 [1]


def step_tables(query_lens: torch.Tensor, context_lens: torch.Tensor, block_tables: torch.Tensor,
                free_blocks: torch.Tensor, free_count: torch.Tensor, num_blocks: int, max_tokens: int,
                block_size: int = 16, out: Optional[StepTables] = None) -> StepTables:
    """The index tensors of one step from request lengths on the GPU (aici_step_tables): what
    BatchInfoBuilder.finish builds on the host from slot lists, without the host.

    Request i has context_lens[i] tokens in the cache and query_lens[i] new ones; `block_tables`
    [requests, max_blocks] names its blocks and is extended in place by the blocks that the new tokens
    begin, taken from the end of `free_blocks[:free_count]`.  `max_tokens` is the size of the token
    tensors (at least the number of new tokens; a captured step takes its largest).  With `out` the
    tensors of an earlier result are written again; out.context_lens may be `context_lens` and
    out.free_count may be `free_count`, which advances the state in place.  A step that does not fit
    (lengths, tokens, free blocks) changes nothing and sets a status bit (see _lib.last_status).  Tokens of a
    block whose id is outside the pool get slot -1, and the bit is set too.  Returns a StepTables."""
    fn = "step_tables"
    given = (query_lens, context_lens, block_tables, free_blocks, free_count)
    index, int32 = _one_gpu(fn, given), torch.int32
    for t in given:
        if t.dtype is not int32:
            raise AiciError("%s: lengths, tables and free list must be int32" % fn)
        if t is not block_tables and not t.is_contiguous():
            raise AiciError("%s: lengths and free list must be contiguous" % fn)
    n = query_lens.numel()
    if query_lens.dim() != 1 or context_lens.shape != query_lens.shape or free_blocks.dim() != 1 or \
            free_count.numel() != 1:
        raise AiciError("%s: query_lens and context_lens must be [requests], free_blocks [blocks], free_count [1]" % fn)
    table, rows = block_tables.shape, block_tables.stride()
    if len(table) != 2 or table[0] != n or rows[1] != 1:
        raise AiciError("%s: block_tables must be [requests, max_blocks] with contiguous rows" % fn)
    if not 0 <= max_tokens < 1 << 30:
        raise AiciError("%s: bad max_tokens %d" % (fn, max_tokens))
    if out is None:
        # one allocation; the token tensors first, each on a 16-byte boundary (a piece costs the host 0.9 us)
        if max_tokens % 2 == 0:
            positions, slots, seqlens, logits, context, count = query_lens.new_empty(
                3 * max_tokens + 3 * n + 2).split_with_sizes((2 * max_tokens, max_tokens, n + 1, n, n, 1))
        else:
            positions, _, slots, seqlens, logits, context, count = query_lens.new_empty(
                3 * max_tokens + 3 * n + 4).split_with_sizes((2 * max_tokens, 2, max_tokens, n + 1, n, n, 1))
        positions = positions.view(torch.int64)
        out = StepTables(seqlens, positions, slots, logits, context, count)
    else:
        for t, count, dtype in ((out.seqlens_q, n + 1, torch.int32), (out.positions, max_tokens, torch.int64),
                                (out.slot_mapping, max_tokens, torch.int32), (out.logit_idxs, n, torch.int32),
                                (out.context_lens, n, torch.int32), (out.free_count, 1, torch.int32)):
            if t.get_device() != index or t.dtype is not dtype or t.numel() != count or not t.is_contiguous():
                raise AiciError("%s: out does not match the call (device, types or sizes)" % fn)
    _call(fn, "aici_step_tables", index, query_lens.data_ptr(), context_lens.data_ptr(), block_tables.data_ptr(),
          free_blocks.data_ptr(), free_count.data_ptr(), n, table[1], rows[0] if n > 1 else table[1],
          free_blocks.numel(), num_blocks, block_size, max_tokens, out.seqlens_q.data_ptr(),
          out.positions.data_ptr(), out.slot_mapping.data_ptr(), out.logit_idxs.data_ptr(),
          out.context_lens.data_ptr(), out.free_count.data_ptr())
    return out
