"""KV cache of one layer held in 8 bits: write, attention, eviction by accumulated attention weight.

``Kv8Cache.tensor`` is a uint8 tensor ``[2 (K, V), num_blocks, record]``; a record holds ``kv_heads x block_size x
head_dim`` e4m3 values and one power-of-two fp32 scale for each head (include/pegaflow_b200.h, section 5).  A cache registers
like any KV tensor whose first dimension is 2 (``PegaWorkerConnector.register_kv_caches({name: cache})``), so that saves, loads
and peer copies move half the bytes of a 16-bit cache and a block's scales travel with it.  Of a cache in a slice of a larger
buffer its records alone are registered, with an engine of the same process; ``cache.tensor`` in its place would be taken to own
all bytes from one block to the next.

The calls only enqueue work, on the current torch stream of the cache's device unless ``stream`` (a cudaStream_t value)
says otherwise, and may be captured into a CUDA graph.  Work on a given stream comes behind what the current stream holds at
the call, and the memory of the call's tensors and outputs is not given out again before either stream is through with
them; to use the outputs, the current stream has to wait for the given one.  (A stream that is being captured while the current
one is not cannot wait for it: order that capture beforehand.)  Block tables, lengths and row starts are int32 tensors on
the device.  What the host cannot check (block ids, lengths, row starts) the kernels check: they leave the access out and
set a bit that ``check()`` raises for.  None of the calls has a backward pass or a forward-mode rule: tensors that carry a derivative are refused.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _native as N

_DTYPES = {torch.bfloat16: N.KV8_BF16, torch.float16: N.KV8_F16}
_INT32, _FLOAT32 = torch.int32, torch.float32
_byref = C.byref
# handle of a device's current stream; torch's own shortcut where there is one, a tenth of the object's cost
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_append, _attention, _attention_workspace, _evict = (N.lib.pf_kv8_append, N.lib.pf_kv8_attention,
                                                     N.lib.pf_kv8_attention_workspace, N.lib.pf_kv8_evict)


def _no_derivative(name, t):
    """Refuses a tensor that autograd would have to know of: neither mode has a rule for these calls."""
    if (t.requires_grad and torch.is_grad_enabled()) or \
            (getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(t).tangent is not None):
        _refuse(f"{name} requires a gradient or carries a tangent: the 8-bit cache has no backward pass and no forward-mode rule")


def _refuse(text: str):
    raise N.PegaflowInvalidArgument(3, "invalid argument: " + text)


class Kv8Cache:
    def __init__(self, num_blocks: int, block_size: int, kv_heads: int, head_dim: int, device="cuda"):
        """A cache of zeros, there when the constructor returns (it waits for the device's current stream, like
        ``from_tensor``).  block_size 16, 32, 64 or 128 tokens, head_dim 64, 128 or 256."""
        record = self.record_bytes(block_size, kv_heads, head_dim)
        self._bind(torch.zeros((2, num_blocks, record), dtype=torch.uint8, device=device), block_size, kv_heads, head_dim)

    @classmethod
    def from_tensor(cls, tensor, block_size: int, kv_heads: int, head_dim: int) -> "Kv8Cache":
        """The cache in an existing uint8 tensor [2, num_blocks, >= record bytes] on a GPU: dense records, at any
        strides that are multiples of 16 bytes (a slice of a buffer that holds several layers, for example)."""
        self = cls.__new__(cls)
        self._bind(tensor, block_size, kv_heads, head_dim)
        return self

    @staticmethod
    def record_bytes(block_size: int, kv_heads: int, head_dim: int) -> int:
        """Bytes of one block of K or of V with its scales."""
        ok = all(isinstance(x, int) and 0 < x < 1 << 31 for x in (block_size, kv_heads, head_dim))
        n = N.lib.pf_kv8_record_bytes(block_size, kv_heads, head_dim) if ok else 0
        if not n:
            _refuse(f"8-bit cache: unsupported geometry block_size={block_size} kv_heads={kv_heads} head_dim={head_dim} "
                    "(block_size 16, 32, 64 or 128; kv_heads 1 to 1024; head_dim 64, 128 or 256)")
        return n

    def _bind(self, t, block_size, kv_heads, head_dim):
        record = self.record_bytes(block_size, kv_heads, head_dim)
        if t.dtype != torch.uint8 or t.dim() != 3 or t.shape[0] != 2 or t.shape[2] < record or t.shape[1] == 0:
            _refuse(f"8-bit cache: a uint8 tensor [2, num_blocks, {record}] is needed, not {t.dtype} {tuple(t.shape)}")
        if not t.is_cuda:
            _refuse(f"8-bit cache: the tensor is on {t.device}, not on a GPU")
        if t.stride(2) != 1 or t.stride(0) < record or (t.shape[1] > 1 and t.stride(1) < record):
            _refuse(f"8-bit cache: records of {record} bytes do not fit the strides {t.stride()}")
        if t.data_ptr() % 16 or t.stride(0) % 16 or (t.shape[1] > 1 and t.stride(1) % 16):
            _refuse("8-bit cache: address and strides must be multiples of 16 bytes")
        self.tensor = t
        self.block_size, self.kv_heads, self.head_dim = block_size, kv_heads, head_dim
        self.num_blocks = t.shape[1]
        self.device = t.device
        self._index = t.device.index
        block_stride = t.stride(1) if t.shape[1] > 1 else -(-record // 16) * 16
        self._desc = N.Kv8CacheDesc(t.data_ptr(), block_stride, t.stride(0), t.shape[1], block_size, kv_heads, head_dim)
        self._desc_ref = _byref(self._desc)
        self._status = torch.zeros(1, dtype=torch.int32, device=t.device)
        # any stream may be the first to use the cache: the status, which nobody else can wait for, is there before that
        with torch.cuda.device(t.device):
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream().synchronize()
        self._status_ptr = self._status.data_ptr()
        self._workspaces = {}      # sizes of a call -> workspace bytes
        n = kv_heads * block_size * head_dim
        #: View of the e4m3 values: [2, num_blocks, kv_heads, block_size, head_dim].
        self.values = t[:, :, :n].view(torch.float8_e4m3fn).view(2, t.shape[1], kv_heads, block_size, head_dim)
        #: View of the scales: [2, num_blocks, kv_heads], float32.
        self.scales = t[:, :, n:n + 4 * kv_heads].view(torch.float32)

    def registration(self):
        """What an engine needs to know of the layer: (tensor, or (address, bytes) where it is a slice of a larger buffer; number
        of blocks; bytes of a segment; from K to V of a block; from block to block, None where blocks are dense)."""
        t = self.tensor
        n, width = t.shape[1], t.shape[2]
        if t.storage_offset() == 0 and t.stride(1) == width:
            return t, n, width, t.stride(0), None
        behind = t.untyped_storage().nbytes() - t.storage_offset()
        record = self.record_bytes(self.block_size, self.kv_heads, self.head_dim)
        return (t.data_ptr(), behind), n, record, t.stride(0), max(t.stride(1), record)

    def check(self):
        """Raise if a call since the last check met a block id, a length or row starts that it had to leave out.  Waits
        for the device's current stream."""
        bits = int(self._status.item())
        if bits:
            self._status.zero_()
            what = [text for bit, text in ((N.KV8_BAD_BLOCK, "a block id outside the cache"),
                                           (N.KV8_BAD_LENGTH, "a length below 0 or above what block tables or weights hold"),
                                           (N.KV8_BAD_ROWS, "row starts that fall, leave the tensors or exceed max_query"),
                                           (N.KV8_STALLED, "a wait inside a kernel ran out: the outputs are not valid"))
                    if bits & bit]
            _refuse("8-bit cache: " + "; ".join(what))

    # ------------------------------------------------------------------ arguments
    def _ints(self, name, t, dim):
        if t.dtype is not _INT32 or t.dim() != dim or t.device != self.device:
            _refuse(f"{name}: an int32 tensor of {dim} dimension(s) on {self.device} is needed, not {t.dtype} "
                    f"{tuple(t.shape)} on {t.device}")
        if t.stride(-1) != 1 and t.shape[-1] > 1:
            _refuse(f"{name}: the last dimension must be dense")
        return t.data_ptr()

    def _batch(self, block_tables, lens, starts):
        tables_ptr = self._ints("block_tables", block_tables, 2)
        lens_ptr = self._ints("lens", lens, 1)
        n, width = block_tables.shape
        if lens.shape[0] != n:
            _refuse(f"block_tables has {n} rows for {lens.shape[0]} lengths")
        ptr = None
        if starts is not None:
            ptr = self._ints("starts", starts, 1)
            if starts.shape[0] != n + 1:
                _refuse(f"starts has {starts.shape[0]} entries for {n} sequences: {n + 1} are needed")
        return N.Kv8Batch(tables_ptr, block_tables.stride(0), width, n, lens_ptr, ptr, self._status_ptr)

    def _rows(self, name, t, heads=None):
        """Checks a tensor of rows; returns its dtype's code and its strides."""
        code = _DTYPES.get(t.dtype)
        if code is None or t.dim() != 3 or t.device != self.device:
            _refuse(f"{name}: a bfloat16 or float16 tensor [rows, heads, {self.head_dim}] on {self.device} is needed, not "
                    f"{t.dtype} {tuple(t.shape)} on {t.device}")
        shape, strides = t.shape, t.stride()
        if shape[2] != self.head_dim or (heads is not None and shape[1] != heads):
            _refuse(f"{name}: shape {tuple(shape)} does not fit kv_heads={self.kv_heads}, head_dim={self.head_dim}")
        if strides[2] != 1:
            _refuse(f"{name}: the last dimension must be dense")
        _no_derivative(name, t)
        return code, strides

    def _per_token(self, name, t, n):
        if t.dtype is not _FLOAT32 or t.dim() != 3 or t.device != self.device or t.shape[0] != n or \
                t.shape[1] != self.kv_heads or (t.stride(2) != 1 and t.shape[2] > 1):
            _refuse(f"{name}: a float32 tensor [{n}, {self.kv_heads}, tokens] on {self.device} with a dense last dimension is "
                    f"needed, not {t.dtype} {tuple(t.shape)} on {t.device}")
        _no_derivative(name, t)

    def _hand_over(self, stream, *tensors):
        """The given stream as torch's, behind the current one and known to the allocator as a user of the call's tensors;
        None where it is the current one."""
        current = torch.cuda.current_stream(self.device)
        if stream == current.cuda_stream:
            return None
        given = torch.cuda.ExternalStream(stream, device=self.device)
        with torch.cuda.stream(given):
            alone = torch.cuda.is_current_stream_capturing()
        with torch.cuda.stream(current):
            alone = alone and not torch.cuda.is_current_stream_capturing()
        if not alone:
            given.wait_stream(current)
        for t in (self.tensor, self._status) + tensors:
            if t is not None:
                t.record_stream(given)
        return given

    def _hand_back(self, outputs):
        """What a call on a given stream has allocated is used on the current one."""
        current = torch.cuda.current_stream(self.device)
        for t in outputs:
            t.record_stream(current)

    # ------------------------------------------------------------------ operators
    def append(self, k, v, block_tables, lens, *, starts=None, stream: Optional[int] = None) -> None:
        """Write new tokens.  k, v: [rows, kv_heads, head_dim]; rows starts[s] .. starts[s + 1] (without starts: an equal
        share of the rows) become tokens lens[s], lens[s] + 1, ... of sequence s.  lens holds the lengths before the call
        and is not changed.  A block takes the scale that its largest magnitude needs; where a new row raises it,
        the block's old rows are rounded anew."""
        code, ks = self._rows("k", k, self.kv_heads)
        v_code, vs = self._rows("v", v, self.kv_heads)
        if code != v_code or k.shape != v.shape:
            _refuse(f"k ({k.dtype} {tuple(k.shape)}) and v ({v.dtype} {tuple(v.shape)}) differ")
        batch = self._batch(block_tables, lens, starts)
        if stream is None:
            stream = _stream_of(self._index)
        else:
            self._hand_over(stream, k, v, block_tables, lens, starts)
        N.check(_append(self._index, self._desc_ref, _byref(batch), k.data_ptr(), v.data_ptr(), code, k.shape[0], ks[0], ks[1],
                        vs[0], vs[1], stream))

    def attention(self, q, block_tables, lens, *, starts=None, max_query: Optional[int] = None,
                  scale: Optional[float] = None, causal: bool = True, weights=None, lse: bool = False, out=None,
                  stream: Optional[int] = None):
        """Attention of q [rows, q_heads, head_dim] over the cache; returns out, or (out, lse) with ``lse=True``.

        lens counts the rows' own tokens, which are in the cache already: row i of a sequence with n rows is
        token lens - n + i and sees, unless ``causal=False``, the tokens up to itself.  A row that sees none
        gives 0 and lse = -inf.  max_query: the most rows of any sequence (needed with starts).  scale: head_dim ** -0.5
        unless given.  weights, float32 [sequences, kv_heads, >= longest]: each token's probability, summed over the
        sequence's rows and the query heads of the KV head, is added in place.  Rows of no sequence, in front of starts[0]
        and behind the last one, are left as they were in a given ``out``, and 0 in one that the call allocates; their
        lse is -inf."""
        code, qs = self._rows("q", q)
        n_rows, q_heads, dim = q.shape
        if q_heads == 0 or q_heads % self.kv_heads:
            _refuse(f"{q_heads} query heads are not a multiple of {self.kv_heads} KV heads")
        batch = self._batch(block_tables, lens, starts)
        if max_query is None:
            if starts is not None:
                _refuse("max_query is needed with starts")
            max_query = n_rows // max(1, batch.n_seqs)
        elif max_query < 0:
            _refuse(f"max_query={max_query}")
        w_ptr, w_seq, w_head, capacity = None, 0, 0, 0
        if weights is not None:
            self._per_token("weights", weights, batch.n_seqs)
            w_ptr, (w_seq, w_head, _), capacity = weights.data_ptr(), weights.stride(), weights.shape[2]
        clear = 0
        if out is not None:
            self._rows("out", out)
            if out.shape != q.shape or out.dtype != q.dtype:
                _refuse(f"out ({out.dtype} {tuple(out.shape)}) and q ({q.dtype} {tuple(q.shape)}) differ")
        if starts is not None and (out is None or lse):        # what the call allocates has no row that nobody writes
            clear = N.KV8_CLEAR_ALL if out is None else N.KV8_CLEAR_LSE
        if stream is not None:
            given = self._hand_over(stream, q, block_tables, lens, starts, weights, out)
            if given is not None:
                with torch.cuda.stream(given):     # what the call allocates belongs to the stream that uses it
                    result = self.attention(q, block_tables, lens, starts=starts, max_query=max_query, scale=scale, causal=causal,
                                            weights=weights, lse=lse, out=out)
                self._hand_back(result if lse else (result,))
                return result
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        os = out.stride()
        lse_out = torch.empty((n_rows, q_heads), dtype=_FLOAT32, device=self.device) if lse else None
        args = N.Kv8AttentionArgs(q.data_ptr(), out.data_ptr(), lse_out.data_ptr() if lse else None, w_ptr, n_rows, max_query,
                                  qs[0], qs[1], os[0], os[1], w_seq, w_head, capacity, q_heads, code, 1 if causal else 0, clear,
                                  dim ** -0.5 if scale is None else scale)
        sizes = (n_rows, q_heads, max_query, batch.n_seqs, batch.max_blocks, starts is None, lse, w_ptr is None, capacity)
        need = self._workspaces.get(sizes)
        if need is None:
            size = N.sz()
            N.check(_attention_workspace(self._index, self._desc_ref, _byref(batch), _byref(args), _byref(size)))
            if len(self._workspaces) >= 1024:
                self._workspaces.clear()
            need = self._workspaces[sizes] = size.value
        space = torch.empty(need, dtype=torch.uint8, device=self.device)
        N.check(_attention(self._index, self._desc_ref, _byref(batch), _byref(args), space.data_ptr(), need,
                           _stream_of(self._index)))
        return (out, lse_out) if lse else out

    def evict(self, block_tables, lens, weights, dst_tables, keep: int, *, recent: int = 0,
              stream: Optional[int] = None) -> Tuple["torch.Tensor", "torch.Tensor", "torch.Tensor"]:
        """Shorten every sequence to at most ``keep`` tokens by accumulated attention weight.

        Of each sequence and KV head the last ``recent`` tokens are kept and, of the others, those of largest weight (equal
        ones: the earlier token), in their order.  They are copied into the blocks of dst_tables [sequences,
        ceil(keep / block_size)], which must not be among block_tables; the source blocks, which other sequences may
        share, are not changed.  weights as ``attention`` accumulates them.

        Returns (lens, weights, kept): int32 [sequences]; float32 like weights, 0 behind the kept tokens, so that
        attention can go on adding; int32 [sequences, kv_heads, keep], the source token of each, -1 behind the last."""
        batch = self._batch(block_tables, lens, None)
        dst_ptr = self._ints("dst_tables", dst_tables, 2)
        n, heads = batch.n_seqs, self.kv_heads
        if not 0 < keep < 1 << 31 or not 0 <= recent <= keep:
            _refuse(f"keep={keep}, recent={recent}: keep must be positive and recent at most keep")
        if dst_tables.shape[0] != n or dst_tables.shape[1] * self.block_size < keep:
            _refuse(f"dst_tables {tuple(dst_tables.shape)} does not hold {keep} tokens of {n} sequences")
        self._per_token("weights", weights, n)
        if stream is not None:
            given = self._hand_over(stream, block_tables, lens, weights, dst_tables)
            if given is not None:
                with torch.cuda.stream(given):
                    result = self.evict(block_tables, lens, weights, dst_tables, keep, recent=recent)
                self._hand_back(result)
                return result
        ws, tokens = weights.stride(), weights.shape[2]
        capacity = max(tokens, keep)
        new_lens = torch.empty(n, dtype=_INT32, device=self.device)
        new_weights = torch.empty((n, heads, capacity), dtype=_FLOAT32, device=self.device)
        kept = torch.empty((n, heads, keep), dtype=_INT32, device=self.device)
        args = N.Kv8EvictArgs(weights.data_ptr(), ws[0], ws[1], tokens, dst_ptr, dst_tables.stride(0), keep, recent,
                              new_lens.data_ptr(), new_weights.data_ptr(), capacity, kept.data_ptr())
        N.check(_evict(self._index, self._desc_ref, _byref(batch), _byref(args),
                       _stream_of(self._index)))
        return new_lens, new_weights, kept
