"""Operators of the softmax-attention layers that stand between linear-attention layers: the plan of a paged cache, rotary
positions, the append to a cache held in 8 bits and the attention that reads it.

The cache is a pool of pages of ``block_size`` tokens (a power of two, 16 .. 256): codes ``[pages, heads, block_size, D]`` in
``torch.float8_e4m3fn`` or ``torch.int8`` with any outer strides (a ``[pages, block_size, heads, D]`` pool is passed as
``pool.transpose(1, 2)``) and fp32 scales ``[pages, heads]``; a stored value is code times scale.  Lengths, tables and
slots are device tensors read by the kernels: no call waits for the GPU, and each may be captured into a graph and replayed
with other contents.  The reference has no counterpart of these operators.
"""
from __future__ import annotations

import ctypes
import functools
import struct

from . import _runtime

_VP, _I64, _F64, _B = ctypes.c_void_p, ctypes.c_int64, ctypes.c_double, ctypes.c_bool

# operands of the C entry points; a tensor is a pointer to a packed fla_tensor
OP_ARGTYPES = {
    "paged_kv_plan": [_VP] * 5 + [_I64] + [_VP] * 6,
    "rotary_axes": [_VP] * 5 + [_B, _B, _VP, _VP],
    "paged_kv_append": [_VP] * 7,
    "paged_kv_attention": [_VP] * 8 + [_F64, _I64, _B, _VP, _VP],
}

# fla_tensor of each rank: pointer, type, rank, extents and strides, each padded to eight
_FLA_TENSOR = tuple(struct.Struct(f"Pii{n}q{8 * (8 - n)}x{n}q{8 * (8 - n)}x") for n in range(_runtime.FLA_MAX_DIMS + 1))
_CODES = {"torch.float32": 0, "torch.float16": 1, "torch.bfloat16": 2, "torch.int32": 3, "torch.int64": 4, "torch.int8": 5,
          "torch.float8_e4m3fn": 6}
_CODE_OF = {}     # torch.dtype -> fla_dtype


class _Call:
    """Packs the tensors of one call as ``fla_tensor`` bytes (ctypes hands their address to the library for the time of
    the call): a tenth of the time that ctypes structures take, which a decode step would otherwise spend on the host."""

    def __init__(self, anchor, name: str):
        if not getattr(anchor, "is_cuda", False):
            _runtime.ensure_gpu_tensor(anchor, name)
        self.device = anchor.device
        self.index = anchor.get_device()

    def tensor(self, t, name: str):
        if t is None:
            return None
        try:
            if t.get_device() == self.index:
                shape = t.shape
                n = len(shape)
                return _FLA_TENSOR[n].pack(t.data_ptr(), _CODE_OF[t.dtype], n, *shape, *t.stride())
        except (AttributeError, KeyError, IndexError):
            pass
        return self._checked(t, name)

    def _checked(self, t, name: str):
        """What is wrong with ``t``; or a type seen for the first time."""
        _runtime.ensure_gpu_tensor(t, name)
        if t.device != self.device:
            raise ValueError(f"{name} must be on {self.device}, got {t.device}; one call cannot mix tensors from different devices.")
        if t.dim() > _runtime.FLA_MAX_DIMS:
            raise ValueError(f"{name} has rank {t.dim()} > {_runtime.FLA_MAX_DIMS}.")
        code = _CODES.get(str(t.dtype))
        if code is None:
            raise TypeError(f"fla_hip: {name} has unsupported tensor dtype {t.dtype}.")
        _CODE_OF[t.dtype] = code
        return self.tensor(t, name)

    def run(self, name: str, *args):
        """``fla_<name>(<operands>, stream)`` on the current stream of the call's device."""
        launch = _runtime.bind_direct(name, OP_ARGTYPES[name])
        if _runtime.is_current(self.index):
            status = launch(*args, _runtime.raw_stream(self.index))
        else:
            with _runtime.device_guard(self.index):
                status = launch(*args, _runtime.raw_stream(self.index))
        if status:
            raise RuntimeError(f"fla_{name} failed with status={status}: {_runtime.last_error()}")

    def run_with_workspace(self, name: str, *args):
        """The two-phase call; the workspace comes from torch's caching allocator on the current stream."""
        import torch

        query, launch = _runtime._bind(name, OP_ARGTYPES[name])
        size = ctypes.c_uint64(0)
        with _runtime.device_guard(self.index):
            status = query(*args, ctypes.byref(size))
            if status:
                raise RuntimeError(f"fla_{name}_get_workspace_size failed with status={status}: {_runtime.last_error()}")
            workspace = torch.empty(size.value, dtype=torch.uint8, device=self.device) if size.value else None
            status = launch(*args, workspace.data_ptr() if workspace is not None else None, size.value, _runtime.raw_stream(self.index))
        if status:
            raise RuntimeError(f"fla_{name} failed with status={status}: {_runtime.last_error()}")


def has_tangent(*tensors) -> bool:
    """Whether one of the tensors (or None) is a dual tensor of forward-mode differentiation."""
    import torch

    ad = torch.autograd.forward_ad
    return ad._current_level >= 0 and any(t is not None and ad.unpack_dual(t).tangent is not None for t in tensors)


def _refuse_grad(op: str, **tensors):
    import torch

    needing = [name for name, t in tensors.items() if getattr(t, "requires_grad", False)] if torch.is_grad_enabled() else []
    if torch.autograd.forward_ad._current_level >= 0:
        needing += [name for name, t in tensors.items() if name not in needing and has_tangent(t)]
    if needing:
        raise NotImplementedError(f"fla_hip.ops.{op}: no gradient is bound for {', '.join(needing)}; pass detached tensors.")


def paged_kv_plan(context_lens, query_lens, block_table, free_blocks, block_size: int, num_tokens: int, *, state_rows=None):
    """Where the tokens of a step go in the cache, in one launch.

    ``context_lens``, ``query_lens`` int32 ``[N]``: tokens each request has in the cache and tokens it adds (0: it sits this
    step out).  ``block_table`` int32 ``[N, M]`` holds each request's pages; the entries of the pages this step opens are
    written, request by request, from ``free_blocks`` int32 ``[F]`` front to back (-1 once the list has run out).
    ``num_tokens``: rows of the step's batch: padded, or cut off (tokens behind it get no slot; ``cu_seqlens`` and
    ``seq_lens`` count them, so that the tokens before keep their places in their requests).  ``state_rows`` int32 ``[N]``: each request's row in a state
    pool.  Returns

    * ``slot_mapping`` int64 ``[num_tokens]``: page * block_size + offset, -1 for a token without a page and for padding,
    * ``positions`` int32 ``[num_tokens]``: position in the request's text, 0 for padding,
    * ``cu_seqlens`` int32 ``[N + 1]``: query rows of each request; ``seq_lens`` int32 ``[N]``: context + query,
    * ``blocks_used`` int32 ``[1]``: entries of ``free_blocks`` needed; more than F means that the list ran out,
    * ``state_indices`` int32 ``[num_tokens]`` (-1 for padding): ``ssm_state_indices`` of ``recurrent_gated_delta_rule``;
      None without ``state_rows``.
    """
    import torch

    call = _Call(block_table, "block_table")
    if block_table.dim() != 2:
        raise ValueError(f"paged_kv_plan: block_table must be [N, M], got rank {block_table.dim()}.")
    if num_tokens < 0:
        raise ValueError(f"paged_kv_plan: num_tokens must not be negative, got {num_tokens}.")
    n, dev, i32 = block_table.shape[0], call.device, torch.int32
    slots = torch.empty(num_tokens, dtype=torch.int64, device=dev)
    # the int32 results are parts of one allocation
    sizes = [num_tokens, n + 1, n, 1] if state_rows is None else [num_tokens, n + 1, n, 1, num_tokens]
    ints = torch.empty(sum(sizes), dtype=i32, device=dev)
    positions, cu, seq, used, *rest = ints.split_with_sizes(sizes)
    states = rest[0] if rest else None
    if n == 0:
        slots.fill_(-1)
        for t in (positions, cu, used):
            t.zero_()
        if states is not None:
            states.fill_(-1)
        return slots, positions, cu, seq, used, states
    d, at = call.tensor, ints.data_ptr()
    new = lambda first, count: _FLA_TENSOR[1].pack(at + 4 * first, _CODES["torch.int32"], 1, count, 1)
    call.run("paged_kv_plan", d(context_lens, "context_lens"), d(query_lens, "query_lens"), d(block_table, "block_table"),
             d(free_blocks, "free_blocks"), d(state_rows, "state_rows"), block_size, d(slots, "slot_mapping"), new(0, num_tokens),
             new(num_tokens, n + 1), new(num_tokens + n + 1, n), new(num_tokens + 2 * n + 1, 1),
             None if states is None else new(num_tokens + 2 * n + 2, num_tokens))
    return slots, positions, cu, seq, used, states


@functools.lru_cache(maxsize=64)
def _axis_table(sections: tuple, axis_order: str):
    """Axis of each frequency as a host array: contiguous sections, or the axes in turn while they have any left.  None for
    sections that make no sense."""
    left, got = list(sections), []
    if any(n < 0 for n in left):
        return None, None
    if axis_order == "blocked":
        got = [a for a, n in enumerate(left) for _ in range(n)]
    else:
        while any(left):
            for a, n in enumerate(left):
                if n:
                    left[a] -= 1
                    got.append(a)
    data = (ctypes.c_int64 * len(got))(*got)
    return data, _runtime.FlaIntArray(ctypes.cast(data, ctypes.POINTER(ctypes.c_int64)), len(got))


def _rotate(q, k, positions, inv_freq, sections, axis_order: str, pairing: str, inverse: bool):
    import torch

    if axis_order not in ("blocked", "interleaved"):
        raise ValueError(f"rotary_axes: axis_order must be 'blocked' or 'interleaved', got {axis_order!r}.")
    if pairing not in ("half", "adjacent"):
        raise ValueError(f"rotary_axes: pairing must be 'half' or 'adjacent', got {pairing!r}.")
    call = _Call(q, "q")
    sections = tuple(map(int, sections))
    table = _axis_table(sections, axis_order)[1]
    if table is None or table.size != inv_freq.numel():
        raise ValueError(f"rotary_axes: sections {sections} must be non-negative and sum to the {inv_freq.numel()} frequencies.")
    if positions.dim() < 1 or positions.shape[0] != len(sections):
        raise ValueError(f"rotary_axes: positions must have one row for each of the {len(sections)} sections.")
    q_out = torch.empty_like(q)
    k_out = None if k is None else torch.empty_like(k)
    if q.numel() == 0 or (k is not None and k.numel() == 0):      # one of the two is empty: the other goes alone
        if q.numel():
            return _rotate(q, None, positions, inv_freq, sections, axis_order, pairing, inverse)[0], k_out
        if k is not None and k.numel():
            return q_out, _rotate(k, None, positions, inv_freq, sections, axis_order, pairing, inverse)[0]
        return q_out, k_out
    d = call.tensor
    call.run("rotary_axes", d(q, "q"), d(k, "k"), d(positions, "positions"), d(inv_freq, "inv_freq"),
             ctypes.addressof(table), pairing == "adjacent", inverse, d(q_out, "q_out"), d(k_out, "k_out"))
    return q_out, k_out


def rotary_axes_fwd(q, k, positions, inv_freq, sections, *, axis_order: str = "blocked", pairing: str = "half"):
    """Rotary positions with one or more axes; see ``rotary_axes``, which binds the gradient."""
    return _rotate(q, k, positions, inv_freq, sections, axis_order, pairing, False)


def rotary_axes_bwd(dq, dk, positions, inv_freq, sections, *, axis_order: str = "blocked", pairing: str = "half"):
    """Gradient of ``rotary_axes_fwd``: the same rotation by the negative angles."""
    return _rotate(dq, dk, positions, inv_freq, sections, axis_order, pairing, True)


def paged_kv_append(key, value, key_cache, value_cache, key_scales, value_scales, slot_mapping):
    """Quantises ``key`` and ``value`` ``[T, H, D]`` into the pages that ``slot_mapping`` int64 ``[T]`` names (negative: the row
    is skipped), as ``paged_kv_plan`` lays them out: the rows of one page are one run, neighbours with slots that ascend by
    one (a page named by two separate runs of rows in one call, or by the same slot twice, has unspecified contents).  A page's scale is the smallest power of
    two ``s`` with ``max|x| / s <= 448`` (e4m3) or ``127`` (int8) over the tokens of that page and head so far; when it grows,
    the codes already there are converted.  Tokens of a page before the first new one are kept; a page whose offset 0 is
    written starts afresh.  Infinities store the largest code; NaN stores NaN (e4m3) or 0 (int8)."""
    _refuse_grad("paged_kv_append", key=key, value=value, key_scales=key_scales, value_scales=value_scales)
    call = _Call(key_cache, "key_cache")
    if key.dim() != 3 or key.shape[0] == 0:
        if key.dim() == 3 and key.shape == value.shape and slot_mapping.numel() == 0:
            return
        raise ValueError(f"paged_kv_append: key and value must be [T, H, D] with one slot for each row, got {tuple(key.shape)}.")
    d = call.tensor
    call.run("paged_kv_append", d(key, "key"), d(value, "value"), d(key_cache, "key_cache"), d(value_cache, "value_cache"),
             d(key_scales, "key_scales"), d(value_scales, "value_scales"), d(slot_mapping, "slot_mapping"))


def paged_kv_attention(query, key_cache, value_cache, key_scales, value_scales, block_table, seq_lens, cu_seqlens=None, *,
                       scale=None, max_query_len=None, return_lse: bool = False, out=None):
    """Softmax attention over the cache: ``query [T, Hq, D]`` (bf16 or fp16; D 64, 128 or 256; Hq a multiple of the cache's
    heads), ``block_table`` int32 ``[N, M]``, ``seq_lens`` int32 ``[N]`` (tokens in the cache, the new ones included),
    ``cu_seqlens`` int32 ``[N + 1]`` the query rows of each request, or None for one row each (decode).  Row j of a
    request's q rows is token ``seq_lens - q + j`` and sees the tokens up to itself, also in a request that goes on behind the
    last row of ``query``; pages that the table gives a number outside the pool are not seen, and a row that sees nothing is 0 with lse -inf.  ``scale`` defaults to ``D ** -0.5``.
    ``max_query_len``: the largest number of query rows of a request, if the caller knows it.  It only chooses the kernel, but
    a batch of few rows each is slower without it (128 requests of one row up to 8192 tokens: 210 us with it, 313 without).
    Rows that belong to no request are 0 in a new result and left as they are in a given ``out``.  Returns ``out`` or, with
    ``return_lse``, ``(out, lse)`` with lse fp32 ``[T, Hq]`` (natural logarithm)."""
    import torch

    _refuse_grad("paged_kv_attention", query=query, key_cache=key_cache, value_cache=value_cache, key_scales=key_scales, value_scales=value_scales)
    call = _Call(query, "query")
    if query.dim() != 3:
        raise ValueError(f"paged_kv_attention: query must be [T, Hq, D], got rank {query.dim()}.")
    clear = out is None
    if clear:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    rows, heads, dim = query.shape
    lse = query.new_empty((rows, heads), dtype=torch.float32) if return_lse else None
    if rows == 0 or block_table.shape[0] == 0:
        if cu_seqlens is None and rows != block_table.shape[0]:
            raise ValueError("paged_kv_attention: without cu_seqlens query must have one row for each request.")
        if clear:
            out.zero_()
        if lse is not None:
            lse.fill_(float("-inf"))
        return (out, lse) if return_lse else out
    if not clear and lse is not None and cu_seqlens is not None:
        lse.fill_(float("-inf"))      # rows behind the last request: `out` stays as it is, lse is new
    d = call.tensor
    q = d(query, "query")
    # descriptors of new results are written down: nothing about them has to be asked
    to = _FLA_TENSOR[3].pack(out.data_ptr(), _CODE_OF[query.dtype], 3, rows, heads, dim, heads * dim, dim, 1) if clear else d(out, "out")
    call.run_with_workspace(
        "paged_kv_attention", q, d(key_cache, "key_cache"), d(value_cache, "value_cache"), d(key_scales, "key_scales"),
        d(value_scales, "value_scales"), d(block_table, "block_table"), d(seq_lens, "seq_lens"), d(cu_seqlens, "cu_seqlens"),
        dim ** -0.5 if scale is None else float(scale), 0 if max_query_len is None else int(max_query_len), clear, to,
        None if lse is None else _FLA_TENSOR[2].pack(lse.data_ptr(), _CODES["torch.float32"], 2, rows, heads, heads, 1))
    return (out, lse) if return_lse else out
