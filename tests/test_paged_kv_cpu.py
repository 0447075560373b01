"""Host-side contract of the paged 8-bit attention operators, without a GPU: what the entry points refuse, workspace sizes,
the front end's checks, and the oracle against closed forms and torch's own 8-bit conversion.  Nothing is launched."""
import ctypes
import math

import pytest
import torch

from oracle import paged_kv as ref

F32, F16, BF16, I32, I64, I8, F8 = range(7)
OK, NULL, DTYPE, SHAPE, UNSUPPORTED, WORKSPACE = range(6)


@pytest.fixture(scope="module")
def lib():
    import fla_hip

    return fla_hip.load_library()


def desc(shape, dtype, strides=None, data=4096):
    """A packed descriptor of memory that is never touched."""
    from fla_hip.ops import _paged_kv as P

    if strides is None:
        strides, n = [], 1
        for d in reversed(shape):
            strides.insert(0, n)
            n *= d
    return P._FLA_TENSOR[len(shape)].pack(data, dtype, len(shape), *shape, *strides)


def test_packed_descriptors_are_the_structure_of_the_header():
    from fla_hip.ops._runtime import FlaTensor

    packed = FlaTensor.from_buffer_copy(desc((2, 3, 5), BF16, (40, 8, 1), data=123456))
    assert (packed.data, packed.dtype, packed.ndim) == (123456, BF16, 3)
    assert list(packed.shape) == [2, 3, 5, 0, 0, 0, 0, 0] and list(packed.stride) == [40, 8, 1, 0, 0, 0, 0, 0]
    assert ctypes.sizeof(FlaTensor) == len(desc((1,), F32)) == len(desc((1,) * 8, F32))


def attention_args(**change):
    a = dict(query=desc((6, 8, 128), BF16), key_cache=desc((10, 2, 16, 128), F8), value_cache=desc((10, 2, 16, 128), F8),
             key_scales=desc((10, 2), F32), value_scales=desc((10, 2), F32), block_table=desc((3, 4), I32), seq_lens=desc((3,), I32),
             cu_seqlens=desc((4,), I32), scale=0.1, max_query_len=3, clear_tail=True, out=desc((6, 8, 128), BF16), lse=desc((6, 8), F32))
    a.update(change)
    return list(a.values())


def query(lib, args):
    from fla_hip.ops import _paged_kv as P

    fn = lib.fla_paged_kv_attention_get_workspace_size
    fn.argtypes, fn.restype = [*P.OP_ARGTYPES["paged_kv_attention"], ctypes.POINTER(ctypes.c_uint64)], ctypes.c_int
    size = ctypes.c_uint64(77)
    return fn(*args, ctypes.byref(size)), size.value, lib.fla_last_error().decode()


@pytest.mark.parametrize("change,status,text", [
    (dict(query=None), NULL, "query must not be null"),
    (dict(query=desc((6, 8, 128), F32)), DTYPE, "query has unsupported dtype"),
    (dict(query=desc((6, 7, 128), BF16), out=desc((6, 7, 128), BF16)), SHAPE, "not a multiple"),
    (dict(query=desc((6, 8, 64), BF16), out=desc((6, 8, 64), BF16)), SHAPE, "query has 64 channels"),
    (dict(query=desc((6, 8, 128), BF16, (1028, 128, 1))), SHAPE, "16-byte aligned"),
    (dict(query=desc((6, 8, 128), BF16, data=4100)), SHAPE, "16-byte aligned"),
    (dict(query=desc((6, 8, 128), BF16, (-1024, 128, 1))), SHAPE, "rows of query"),
    (dict(out=desc((6, 8, 128), F16)), DTYPE, "out has unsupported dtype"),
    (dict(out=desc((6, 8, 128), BF16, (0, 128, 1))), SHAPE, "rows of out overlap"),
    (dict(out=desc((5, 8, 128), BF16)), SHAPE, "shape of query"),
    (dict(key_cache=desc((10, 2, 16, 128), BF16)), DTYPE, "key_cache has unsupported dtype"),
    (dict(value_cache=desc((10, 2, 16, 128), I8)), SHAPE, "same shape and type"),
    (dict(key_cache=desc((10, 2, 24, 128), F8), value_cache=desc((10, 2, 24, 128), F8)), UNSUPPORTED, "power of two from 16 to 256"),
    (dict(key_cache=desc((10, 2, 8, 128), F8), value_cache=desc((10, 2, 8, 128), F8)), UNSUPPORTED, "power of two from 16 to 256"),
    (dict(key_cache=desc((10, 2, 16, 96), F8), value_cache=desc((10, 2, 16, 96), F8)), UNSUPPORTED, "head size must be"),
    (dict(key_cache=desc((10, 2, 16, 128), F8, (4096, 2048, 136, 1))), SHAPE, "16-byte aligned"),
    (dict(key_cache=desc((10, 2, 16, 128), F8, (4096, 2048, 1, 16))), SHAPE, "rows of key_cache must be contiguous"),
    (dict(key_cache=desc((10, 2, 16, 128), F8, (4096, 2048, 1 << 23, 1))), UNSUPPORTED, "too far apart"),
    (dict(key_scales=desc((10, 3), F32)), SHAPE, "key_scales must be"),
    (dict(value_scales=desc((10, 2), BF16)), DTYPE, "value_scales has unsupported dtype"),
    (dict(block_table=desc((3, 4), I64)), DTYPE, "block_table has unsupported dtype"),
    (dict(block_table=desc((3, 4), I32, (4, 2))), SHAPE, "unit innermost stride"),
    (dict(block_table=desc((3, 1 << 28), I32)), SHAPE, "more than 2^31"),
    (dict(seq_lens=desc((4,), I32)), SHAPE, "seq_lens must be"),
    (dict(cu_seqlens=desc((3,), I32)), SHAPE, "cu_seqlens must be"),
    (dict(cu_seqlens=None), SHAPE, "one row for each of the 3 requests"),
    (dict(lse=desc((6, 7), F32)), SHAPE, "lse must be"),
    (dict(max_query_len=-1), SHAPE, "must not be negative"),
])
def test_attention_refusals(lib, change, status, text):
    got, _, message = query(lib, attention_args(**change))
    assert got == status and text in message, (got, message)


def test_attention_workspace(lib):
    """Nothing for one chunk to a tile; else room for 2048 / heads items beyond the tiles, each of heads x rows x (D + 2) fp32."""
    assert query(lib, attention_args())[:2] == (OK, 0)                       # the table names 64 tokens
    wide = dict(block_table=desc((3, 1000), I32))
    status, size, _ = query(lib, attention_args(**wide))
    tiles = 6 * 4 // 16 + 3                                                   # 6 rows of 4 heads in tiles of 16, at most one more each
    assert status == OK and size == (tiles + 256) * 2 * 16 * (128 + 2) * 4
    assert query(lib, attention_args(**wide, cu_seqlens=None, query=desc((3, 8, 128), BF16), out=desc((3, 8, 128), BF16), lse=None))[1] == (3 + 256) * 2 * 16 * 130 * 4
    assert query(lib, attention_args(lse=None))[0] == OK
    from fla_hip.ops import _paged_kv as P

    fn = lib.fla_paged_kv_attention
    fn.argtypes, fn.restype = [*P.OP_ARGTYPES["paged_kv_attention"], ctypes.c_void_p, ctypes.c_uint64, ctypes.c_void_p], ctypes.c_int
    assert fn(*attention_args(**wide), 4096, size - 1, None) == WORKSPACE     # refused before any launch
    assert fn(*attention_args(**wide), None, size, None) == WORKSPACE


def plan_args(**change):
    a = dict(context=desc((3,), I32), query=desc((3,), I32), table=desc((3, 4), I32), free=desc((5,), I32), rows=desc((3,), I32), block=16,
             slots=desc((7,), I64), positions=desc((7,), I32), cu=desc((4,), I32), seq=desc((3,), I32), used=desc((1,), I32), states=desc((7,), I32))
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,status,text", [
    (dict(table=None), NULL, "block_table must not be null"),
    (dict(table=desc((3, 4), I32, (2, 1))), SHAPE, "rows that do not overlap"),
    (dict(context=desc((2,), I32)), SHAPE, "context_lens must have 3"),
    (dict(query=desc((3,), I64)), DTYPE, "query_lens has unsupported dtype"),
    (dict(query=desc((3,), I32, (2,))), SHAPE, "query_lens must be contiguous"),
    (dict(free=None), NULL, "free_blocks"),
    (dict(block=48), UNSUPPORTED, "power of two"),
    (dict(slots=desc((7,), I32)), DTYPE, "slot_mapping has unsupported dtype"),
    (dict(positions=desc((6,), I32)), SHAPE, "positions must have 7"),
    (dict(cu=desc((3,), I32)), SHAPE, "cu_seqlens must have 4"),
    (dict(states=None), NULL, "go together"),
    (dict(rows=desc((2,), I32)), SHAPE, "state_rows must have 3"),
])
def test_plan_refusals(lib, change, status, text):
    from fla_hip.ops import _paged_kv as P

    fn = lib.fla_paged_kv_plan
    fn.argtypes, fn.restype = [*P.OP_ARGTYPES["paged_kv_plan"], ctypes.c_void_p], ctypes.c_int
    assert fn(*plan_args(**change), None) == status and text in lib.fla_last_error().decode()


def append_args(**change):
    a = dict(key=desc((5, 2, 128), BF16), value=desc((5, 2, 128), BF16), kc=desc((10, 2, 16, 128), I8), vc=desc((10, 2, 16, 128), I8),
             ks=desc((10, 2), F32), vs=desc((10, 2), F32), slots=desc((5,), I64))
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,status,text", [
    (dict(key=desc((5, 3, 128), BF16)), SHAPE, "key must be [T,2,128]"),
    (dict(value=desc((4, 2, 128), BF16)), SHAPE, "value must be"),
    (dict(value=desc((5, 2, 128), F16)), DTYPE, "value has unsupported dtype"),
    (dict(key=desc((5, 2, 128), BF16, (256, 130, 1))), SHAPE, "16-byte aligned"),
    (dict(key=desc((5, 2, 128), BF16, (1 << 21, 128, 1))), UNSUPPORTED, "too far apart"),
    (dict(slots=desc((5,), I32)), DTYPE, "slot_mapping has unsupported dtype"),
    (dict(slots=desc((4,), I64)), SHAPE, "one slot for each row"),
    (dict(vc=desc((10, 2, 16, 128), F8)), SHAPE, "same shape and type"),
    (dict(kc=desc((0, 2, 16, 128), I8), vc=desc((0, 2, 16, 128), I8), ks=desc((0, 2), F32), vs=desc((0, 2), F32)), SHAPE, "at least one page"),
])
def test_append_refusals(lib, change, status, text):
    from fla_hip.ops import _paged_kv as P

    fn = lib.fla_paged_kv_append
    fn.argtypes, fn.restype = [*P.OP_ARGTYPES["paged_kv_append"], ctypes.c_void_p], ctypes.c_int
    assert fn(*append_args(**change), None) == status and text in lib.fla_last_error().decode()


def rotary_args(axes=(0, 0, 1, 1), **change):
    from fla_hip.ops._runtime import FlaIntArray

    data = (ctypes.c_int64 * len(axes))(*axes)
    table = FlaIntArray(ctypes.cast(data, ctypes.POINTER(ctypes.c_int64)), len(axes))
    a = dict(q=desc((5, 2, 16), BF16), k=desc((5, 1, 16), BF16), positions=desc((2, 5), I64), inv=desc((4,), F32), table=ctypes.addressof(table),
             adjacent=False, inverse=False, q_out=desc((5, 2, 16), BF16), k_out=desc((5, 1, 16), BF16))
    a.update(change)
    return list(a.values()), (data, table)


@pytest.mark.parametrize("axes,change,status,text", [
    ((0, 0, 1, 2), {}, SHAPE, "names axis 2 of 2"),
    ((0, 0, 1), {}, SHAPE, "one entry for each frequency"),
    ((0,) * 9, dict(inv=desc((9,), F32)), SHAPE, "at most half as many"),
    ((0, 0, 1, 1), dict(q=desc((5, 16), BF16)), SHAPE, "must be [B,T,H,D]"),
    ((0, 0, 1, 1), dict(q=desc((5, 2, 16), I32)), DTYPE, "q has unsupported dtype"),
    ((0, 0, 1, 1), dict(k=desc((5, 1, 16), F16)), DTYPE, "k has unsupported dtype"),
    ((0, 0, 1, 1), dict(k=desc((4, 1, 16), BF16), k_out=desc((4, 1, 16), BF16)), SHAPE, "number of heads only"),
    ((0, 0, 1, 1), dict(q=desc((5, 2, 16), BF16, (64, 32, 2))), SHAPE, "unit innermost stride"),
    ((0, 0, 1, 1), dict(q_out=desc((5, 2, 16), BF16, (0, 16, 1))), SHAPE, "rows of an output overlap"),
    ((0, 0, 1, 1), dict(q_out=desc((5, 3, 16), BF16)), SHAPE, "another shape"),
    ((0, 0, 1, 1), dict(k_out=None), NULL, "go together"),
    ((0, 0, 1, 1), dict(positions=desc((2, 6), I64)), SHAPE, "positions must be"),
    ((0, 0, 1, 1), dict(positions=desc((2, 5), F32)), DTYPE, "positions has unsupported dtype"),
    ((0, 0, 1, 1), dict(inv=desc((4,), F32, (2,))), SHAPE, "inv_freq must be contiguous"),
    ((0,), dict(q=desc((5, 2, 15), BF16), q_out=desc((5, 2, 15), BF16), k=None, k_out=None, inv=desc((1,), F32)), SHAPE, "must be even"),
])
def test_rotary_refusals(lib, axes, change, status, text):
    from fla_hip.ops import _paged_kv as P

    fn = lib.fla_rotary_axes
    fn.argtypes, fn.restype = [*P.OP_ARGTYPES["rotary_axes"], ctypes.c_void_p], ctypes.c_int
    args, keep = rotary_args(axes, **change)
    assert fn(*args, None) == status and text in lib.fla_last_error().decode(), lib.fla_last_error()


def test_front_end_refuses_cpu_tensors_and_bad_arguments():
    from fla_hip import ops
    from fla_hip.ops import _paged_kv as P

    x = torch.zeros(2, 1, 64)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(TypeError, match="ROCm GPU tensor"):
        ops.rotary_axes(x, None, i[None], torch.ones(4), (4,))
    with pytest.raises(TypeError, match="ROCm GPU tensor"):
        ops.paged_kv_plan(i, i, torch.zeros(2, 1, dtype=torch.int32), i, 16, 2)
    with pytest.raises(TypeError, match="ROCm GPU tensor"):
        ops.paged_kv_attention(x, x, x, x, x, i, i)
    with pytest.raises(TypeError, match="ROCm GPU tensor"):
        ops.paged_kv_append(x, x, x, x, x, x, i)
    with pytest.raises(ValueError, match="axis_order must be"):
        ops.rotary_axes(x, None, i[None], torch.ones(4), (4,), axis_order="mixed")
    with pytest.raises(ValueError, match="pairing must be"):
        ops.rotary_axes(x, None, i[None], torch.ones(4), (4,), pairing="none")
    with pytest.raises(RuntimeError, match="paged_kv_append mutates key_cache in place"):
        ops.paged_kv_append(x, x, x.clone().requires_grad_(), x, x, x, i)
    with pytest.raises(RuntimeError, match="paged_kv_attention mutates out in place"):
        ops.paged_kv_attention(x, x, x, x, x, i, i, out=x.clone().requires_grad_())
    assert ops.MUTATED_ARGUMENTS["paged_kv_plan"] == ("block_table",)
    assert [list(P._axis_table((3, 2, 1), o)[0]) for o in ("blocked", "interleaved")] == [[0, 0, 0, 1, 1, 2], [0, 1, 2, 0, 1, 0]]
    for name in ("paged_kv_plan", "paged_kv_append", "paged_kv_attention", "rotary_axes", "rotary_axes_fwd", "rotary_axes_bwd"):
        assert name in ops.__all__ and callable(getattr(ops, name))


def test_mutation_guard_finds_arguments_by_place_and_by_name():
    from fla_hip import ops

    seen = []
    guarded = ops._wrap_mutable_op("paged_kv_attention", lambda query, a, b, *, scale=None, out=None: seen.append((query, a, b, scale, out)) or "done")
    out = torch.zeros(3)
    assert guarded(1, 2, b=3, out=out) == "done" and out._version == 1 and seen[-1][2] == 3
    assert guarded(1, 2, 3) == "done" and out._version == 1
    with torch.inference_mode():
        made = torch.zeros(3)
    assert guarded(1, 2, 3, out=made) == "done"                               # no version counter to raise
    by_place = ops._wrap_mutable_op("paged_kv_plan", lambda context, query, block_table, free: None)
    by_place(1, 2, out, 4)
    by_place(1, 2, block_table=out, free=4)
    assert out._version == 3
    with pytest.raises(TypeError):
        by_place(1, 2)
    with pytest.raises(RuntimeError, match="mutates block_table"):
        by_place(1, 2, torch.zeros(2, requires_grad=True), 4)


# ---- the oracle ------------------------------------------------------------------------------------------------------

def test_oracle_codes_are_torch_conversions():
    x = torch.cat([torch.randn(4000, dtype=torch.float64) * s for s in (1e-3, 0.1, 10, 300)] + [torch.tensor([0.0, 447.9, 448, 1e9, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -6], dtype=torch.float64)])
    x = x.float().double()
    want = x.clamp(-448, 448).float().to(torch.float8_e4m3fn).double()
    assert torch.equal(ref.encode(x, torch.float8_e4m3fn), want)
    assert ref.encode(torch.tensor([math.nan, math.inf, -math.inf], dtype=torch.float64), torch.float8_e4m3fn)[1:].tolist() == [448, -448]
    assert ref.encode(torch.tensor([0.5, 1.5, -2.5, 200, math.nan], dtype=torch.float64), torch.int8).tolist() == [0, 2, -2, 127, 0]


@pytest.mark.parametrize("dtype,most", [(torch.float8_e4m3fn, 448.0), (torch.int8, 127.0)])
def test_oracle_scale_is_the_smallest_power_of_two(dtype, most):
    assert ref.step_for(0.0, dtype) == 0 and ref.step_for(most, dtype) == 1 and ref.step_for(most * 1.0000001, dtype) == 2
    for a in (1e-30, 0.37, 5.0, 3e38):
        s = ref.step_for(a, dtype)
        assert math.frexp(s)[0] == 0.5 and a / s <= most < a / (s / 2)


def test_oracle_append_is_one_pass_over_a_page_in_pieces():
    """Powers of two: filling a page row by row in e4m3 gives the codes of the whole page at once (normals)."""
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(16, 1, 64, generator=gen) + torch.sign(torch.randn(16, 1, 64, generator=gen))     # no subnormal codes
    whole, step = torch.zeros(1, 1, 16, 64, dtype=torch.float64), torch.zeros(1, 1, dtype=torch.float64)
    ref.append(x, whole, step, range(16), torch.float8_e4m3fn)
    rows, by_row = torch.zeros_like(whole), torch.zeros_like(step)
    for t in range(16):
        ref.append(x[t:t + 1], rows, by_row, [t], torch.float8_e4m3fn)
    assert torch.equal(whole, rows) and torch.equal(step, by_row)
    assert float((whole[0, 0] * step[0, 0] - x[:, 0]).abs().max() / x.abs().max()) <= 2.0 ** -4


def test_oracle_attention_is_softmax_attention():
    gen = torch.Generator().manual_seed(1)
    kc, vc = torch.randn(4, 2, 16, 64, generator=gen, dtype=torch.float64), torch.randn(4, 2, 16, 64, generator=gen, dtype=torch.float64)
    ks, vs = torch.rand(4, 2, generator=gen), torch.rand(4, 2, generator=gen)
    q = torch.randn(5, 4, 64, generator=gen)
    table = torch.tensor([[2, 0, 3]])
    out, lse, spread, *_ = ref.attention(q, kc, vc, ks, vs, table, [37], [0, 5], 0.125)
    k = (kc * ks.double()[..., None, None])[[2, 0, 3]].transpose(1, 2).flatten(0, 1)[:37].transpose(0, 1).repeat_interleave(2, 0)
    v = (vc * vs.double()[..., None, None])[[2, 0, 3]].transpose(1, 2).flatten(0, 1)[:37].transpose(0, 1).repeat_interleave(2, 0)
    mask = torch.arange(37) <= torch.arange(32, 37)[:, None]
    want = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(0, 1), k, v, attn_mask=mask, scale=0.125)
    assert torch.allclose(out, want.transpose(0, 1), atol=1e-12) and bool((spread >= out.abs() - 1e-12).all())
    score = (q.double().transpose(0, 1) @ k.transpose(-1, -2) * 0.125).masked_fill(~mask, -math.inf)
    assert torch.allclose(lse, score.logsumexp(-1).t(), atol=1e-12)


def test_oracle_rotary_keeps_norms_and_relative_angles():
    gen = torch.Generator().manual_seed(2)
    x, inv = torch.randn(7, 2, 12, generator=gen), torch.rand(5, generator=gen)
    pos = torch.randint(0, 99, (2, 7), generator=gen)
    for order in ("blocked", "interleaved"):
        for pairing in ("half", "adjacent"):
            y = ref.rotary(x, pos, inv, (3, 2), order, pairing)
            assert torch.allclose(y.norm(dim=-1), x.double().norm(dim=-1)) and torch.equal(y[..., 10:], x[..., 10:].double())
            back = ref.rotary(y, pos, inv, (3, 2), order, pairing, inverse=True)
            assert torch.allclose(back, x.double(), atol=1e-12)
            a, b = ref.rotary(x, pos + 5, inv, (3, 2), order, pairing), ref.rotary(x.flip(0), pos + 5, inv, (3, 2), order, pairing)
            assert torch.allclose((a * b).sum(-1), (y * ref.rotary(x.flip(0), pos, inv, (3, 2), order, pairing)).sum(-1))


def test_oracle_plan_closed_form():
    table = [[4, -1], [7, -1]]
    got = ref.plan([16, 3], [2, 15], table, [9, 8], 16, 18, [5, 6])
    assert got["slots"].tolist() == [9 * 16, 9 * 16 + 1] + list(range(7 * 16 + 3, 7 * 16 + 16)) + [8 * 16, 8 * 16 + 1, -1]
    assert got["table"].tolist() == [[4, 9], [7, 8]] and got["used"].tolist() == [2] and got["states"].tolist() == [5, 5] + [6] * 15 + [-1]


@pytest.mark.parametrize("change,text", [
    (dict(kc=desc((10, 2, 16, 128), I8, (4096, 0, 128, 1))), "rows of key_cache overlap"),
    (dict(vc=desc((10, 2, 16, 128), I8, (0, 2048, 128, 1))), "rows of value_cache overlap"),
    (dict(vs=desc((10, 2), F32, (0, 1))), "elements of value_scales overlap"),
    (dict(key=desc((1 << 26, 2, 128), BF16), value=desc((1 << 26, 2, 128), BF16), slots=desc((1 << 26,), I64)), "too many tokens"),
])
def test_append_refuses_caches_that_overlap_and_too_many_tokens(lib, change, text):
    from fla_hip.ops import _paged_kv as P

    fn = lib.fla_paged_kv_append
    fn.argtypes, fn.restype = [*P.OP_ARGTYPES["paged_kv_append"], ctypes.c_void_p], ctypes.c_int
    assert fn(*append_args(**change), None) == SHAPE and text in lib.fla_last_error().decode()


def test_grids_beyond_the_launch_limit_are_refused(lib):
    n = 1 << 23                                         # times two heads of 256 threads: 2^32
    big = dict(query=desc((n, 8, 128), BF16), out=desc((n, 8, 128), BF16), lse=None, block_table=desc((n, 4), I32), seq_lens=desc((n,), I32),
               cu_seqlens=None)
    status, _, text = query(lib, attention_args(**big))
    assert status == SHAPE and "too many query rows" in text
    from fla_hip.ops import _paged_kv as P

    tokens = 1 << 26                                    # four to a workgroup of 256 threads: 2^32
    args, keep = rotary_args(q=desc((tokens, 2, 16), BF16), q_out=desc((tokens, 2, 16), BF16), k=None, k_out=None, positions=desc((2, tokens), I64))
    fn = lib.fla_rotary_axes
    fn.argtypes, fn.restype = [*P.OP_ARGTYPES["rotary_axes"], ctypes.c_void_p], ctypes.c_int
    assert fn(*args, None) == SHAPE and "too many tokens" in lib.fla_last_error().decode()


def test_rotary_refuses_frequencies_that_want_a_gradient():
    from fla_hip import ops

    q, freq = torch.zeros(5, 2, 16, dtype=torch.bfloat16), torch.ones(4, requires_grad=True)
    with pytest.raises(NotImplementedError, match="no gradient is bound for inv_freq"):
        ops.rotary_axes(q, None, torch.zeros(1, 5, dtype=torch.int64), freq, (4,))


@pytest.fixture
def plain_rotary(monkeypatch):
    """``rotary_axes`` with the oracle in the place of the launch."""
    from fla_hip.ops import _paged_kv as P

    def rotate(q, k, positions, inv_freq, sections, axis_order, pairing, inverse):
        assert q.stride(-1) == 1
        return tuple(None if x is None else ref.rotary(x.detach(), positions, inv_freq, sections, axis_order, pairing, inverse).to(x.dtype) for x in (q, k))

    monkeypatch.setattr(P, "_rotate", rotate)


@pytest.mark.parametrize("pairing", ["half", "adjacent"])
def test_rotary_has_a_tangent(plain_rotary, pairing):
    """Linear in q and k: the tangent is the operator applied to the tangents.  Also under a reverse pass, in its gradient, and where
    only one of q and k has one."""
    from fla_hip import ops
    from torch.autograd import forward_ad as ad

    gen = torch.Generator().manual_seed(3)
    q, tq, wq = (torch.randn(5, 3, 12, generator=gen, dtype=torch.float64) for _ in range(3))
    k, tk, wk = (torch.randn(5, 1, 12, generator=gen, dtype=torch.float64) for _ in range(3))
    pos, freq = torch.randint(0, 50, (2, 5), generator=gen), torch.rand(4, generator=gen)
    turn = lambda a, b=None: ops.rotary_axes(a, b, pos, freq, (3, 1), pairing=pairing)
    back = lambda x: ref.rotary(x, pos, freq, (3, 1), "blocked", pairing, True)
    want = turn(tq, tk)
    tangent = lambda x: ad.unpack_dual(x).tangent
    with ad.dual_level():
        a, b = turn(ad.make_dual(q, tq), ad.make_dual(k, tk))
        assert torch.equal(tangent(a), want[0]) and torch.equal(tangent(b), want[1]) and torch.equal(ad.unpack_dual(a).primal, turn(q)[0])
        a, b = turn(ad.make_dual(q, tq), k)
        assert torch.equal(tangent(a), want[0]) and (tangent(b) is None or not bool(tangent(b).any()))
        a, b = turn(q, ad.make_dual(k, tk))
        assert torch.equal(tangent(b), want[1]) and (tangent(a) is None or not bool(tangent(a).any()))
        a, none = turn(ad.make_dual(q, tq))
        assert none is None and torch.equal(tangent(a), want[0])
        with torch.no_grad():
            assert torch.equal(tangent(turn(ad.make_dual(q, tq))[0]), want[0])
        leaf, direction = q.clone().requires_grad_(), tq.clone().requires_grad_()      # both modes at once
        a, _ = turn(ad.make_dual(leaf, direction))
        assert torch.equal(tangent(a), want[0])
        assert torch.equal(torch.autograd.grad(tangent(a), direction, wq, retain_graph=True)[0], back(wq))
        got = torch.autograd.grad(a, leaf, ad.make_dual(wq, tq))[0]                    # the gradient has a tangent too
        assert torch.equal(ad.unpack_dual(got).primal, back(wq)) and torch.equal(tangent(got), back(tq))
    got = torch.autograd.grad(turn(leaf, k.requires_grad_()), (leaf, k), (wq, wk.expand_as(k)))
    assert torch.equal(got[0], back(wq)) and torch.equal(got[1], back(wk))
    assert torch.autograd.gradcheck(lambda x, y: turn(x, y), (leaf, k), check_forward_ad=True)


def test_derivatives_that_are_not_bound_are_refused():
    """Whatever enters the result: queries, caches, scales, frequencies; by gradient and by tangent."""
    from fla_hip import ops
    from torch.autograd import forward_ad as ad

    x, i = torch.zeros(2, 1, 64), torch.zeros(2, dtype=torch.int32)
    cache, scale = torch.zeros(2, 1, 16, 64).to(torch.float8_e4m3fn), torch.zeros(2, 1)
    attention = dict(query=x, key_cache=cache, value_cache=cache, key_scales=scale, value_scales=scale)
    append = dict(key=x, value=x, key_cache=cache, value_cache=cache, key_scales=scale, value_scales=scale)
    for name in attention:
        changed = attention | {name: attention[name].clone().requires_grad_()}
        with pytest.raises(NotImplementedError, match=f"paged_kv_attention: no gradient is bound for {name}"):
            ops.paged_kv_attention(**changed, block_table=i[:, None], seq_lens=i)
        with torch.no_grad(), pytest.raises(TypeError, match="ROCm GPU tensor"):       # no derivative is asked for
            ops.paged_kv_attention(**changed, block_table=i[:, None], seq_lens=i)
    for name in ("key", "value"):
        with pytest.raises(NotImplementedError, match=f"paged_kv_append: no gradient is bound for {name}"):
            ops.paged_kv_append(**append | {name: x.clone().requires_grad_()}, slot_mapping=i.long())
    with ad.dual_level():
        for op, args, rest in ((ops.paged_kv_attention, attention, dict(block_table=i[:, None], seq_lens=i)), (ops.paged_kv_append, append, dict(slot_mapping=i.long()))):
            for name in args:
                if not name.endswith("cache"):
                    with pytest.raises(NotImplementedError, match=f"no gradient is bound for {name}"), torch.no_grad():
                        op(**args | {name: ad.make_dual(args[name], torch.ones_like(args[name]))}, **rest)
        with pytest.raises(NotImplementedError, match="no gradient is bound for inv_freq"):
            ops.rotary_axes(x, None, i[None], ad.make_dual(torch.ones(4), torch.ones(4)), (4,))


@pytest.mark.parametrize("change,text", [
    (dict(kc=desc((10, 2, 16, 128), I8, (2048, 2048, 128, 1))), "rows of key_cache overlap"),        # pages one head apart
    (dict(vc=desc((10, 2, 16, 128), I8, (4096, 2048, 64, 1))), "rows of value_cache overlap"),       # tokens half a row apart
    (dict(kc=desc((10, 2, 16, 128), I8, (4096, 16, 128, 1))), "rows of key_cache overlap"),
    (dict(kc=desc((10, 2, 16, 128), I8, (2032, 1 << 20, 128, 1))), "rows of key_cache overlap"),     # the last row of a page is the next one's
    (dict(ks=desc((10, 2), F32, (1, 1))), "elements of key_scales overlap"),
    (dict(vs=desc((10, 2), F32, (1, 9))), "elements of value_scales overlap"),
    (dict(vc=desc((10, 2, 16, 128), I8, data=4096)), "caches and scales of their own"),
    (dict(ks=desc((10, 2), F32, data=8192), vs=desc((10, 2), F32, data=8192), vc=desc((10, 2, 16, 128), I8, data=1 << 20)), "caches and scales of their own"),
])
def test_append_refuses_memory_that_two_rows_share(lib, change, text):
    """Two workgroups would write it in no order; nothing is launched."""
    from fla_hip.ops import _paged_kv as P

    fn = lib.fla_paged_kv_append
    fn.argtypes, fn.restype = [*P.OP_ARGTYPES["paged_kv_append"], ctypes.c_void_p], ctypes.c_int
    assert fn(*append_args(**change), None) == SHAPE and text in lib.fla_last_error().decode(), lib.fla_last_error()


@pytest.mark.parametrize("change,text", [
    (dict(out=desc((6, 8, 128), BF16, (128, 128, 1))), "rows of out overlap"),
    (dict(out=desc((6, 8, 128), BF16, (1024, 64, 1))), "rows of out overlap"),
    (dict(lse=desc((6, 8), F32, (0, 1))), "elements of lse overlap"),
    (dict(lse=desc((6, 8), F32, (7, 1))), "elements of lse overlap"),
])
def test_attention_refuses_results_that_two_rows_share(lib, change, text):
    assert query(lib, attention_args(**change))[0] == SHAPE and text in lib.fla_last_error().decode()
    nested = dict(out=desc((6, 8, 128), BF16, (128, 1024, 1)), lse=desc((6, 8), F32, (1, 6)))       # heads first: nothing shared
    assert query(lib, attention_args(**nested))[0] == OK


def test_rotary_refuses_results_that_two_rows_share(lib):
    from fla_hip.ops import _paged_kv as P

    fn = lib.fla_rotary_axes
    fn.argtypes, fn.restype = [*P.OP_ARGTYPES["rotary_axes"], ctypes.c_void_p], ctypes.c_int
    for out in (dict(q_out=desc((5, 2, 16), BF16, (16, 16, 1))), dict(k_out=desc((5, 1, 16), BF16, (8, 16, 1)))):
        args, keep = rotary_args(**out)
        assert fn(*args, None) == SHAPE and "rows of an output overlap" in lib.fla_last_error().decode()


def test_a_table_without_columns_needs_no_memory(lib):
    status, size, text = query(lib, attention_args(block_table=desc((3, 0), I32, data=0)))
    assert (status, size) == (OK, 0), text
    assert query(lib, attention_args(block_table=desc((3, 0), I64, data=0)))[0] == NULL
    assert query(lib, attention_args(block_table=desc((3, 4), I32, data=0)))[0] == NULL


def test_strides_of_extents_of_one_may_be_anything(lib):
    one = dict(query=desc((1, 8, 128), BF16, (3, 128, 1)), out=desc((1, 8, 128), BF16, (1, 128, 1)), lse=desc((1, 8), F32, (0, 1)),
               key_cache=desc((1, 2, 16, 128), F8, (5, 2048, 128, 1)), value_cache=desc((1, 2, 16, 128), F8, (0, 2048, 128, 1)),
               key_scales=desc((1, 2), F32, (0, 1)), value_scales=desc((1, 2), F32, (1, 1)))
    status, _, text = query(lib, attention_args(**one))
    assert status == OK, text
    single = dict(query=desc((6, 4, 64), BF16), out=desc((6, 4, 64), BF16), lse=None, key_cache=desc((10, 1, 16, 64), F8, (1024, 1, 64, 1)),
                  value_cache=desc((10, 1, 16, 64), F8, (1024, 1 << 40, 64, 1)), key_scales=desc((10, 1), F32), value_scales=desc((10, 1), F32))
    status, _, text = query(lib, attention_args(**single))
    assert status == OK, text
    assert query(lib, attention_args(query=desc((1, 8, 128), BF16, (3, 64, 1)), out=desc((1, 8, 128), BF16, (3, 64, 1))))[0] == SHAPE
