"""Refusals of the paged-step kernels (PagedBatchBuild, PagedQKVScatter,
PagedAttention, Sample), checked before anything touches a device."""
import pytest

import popcorn_b200 as pc

E = pc.PopcornError
D = pc.DataType
_next = [0x7F0000000000]


def fake(shape, dtype=D.i32, ptr=None):
    """A descriptor over an address range of its own (never dereferenced)."""
    if ptr is None:
        ptr = _next[0]
        n = 1
        for d in shape:
            n *= d
        _next[0] += (n * 8 + 4095) // 4096 * 4096 + 4096
    return pc.Tensor(ptr, shape, dtype)


def refused(code, fn, **kw):
    with pytest.raises(pc.PopcornError) as e:
        fn(**kw)
    assert e.value.code == code, e.value.message
    assert e.value.message


def batch_args(**kw):
    R, W, F, T = 5, 7, 40, 64
    a = dict(cached=fake([R]), added=fake([R]), free_pages=fake([F]), free_head=fake([1]), block_table=fake([R, W]),
             page_size=16, seq_lens=fake([R]), query_start=fake([R + 1]), positions=fake([T]), slots=fake([T]),
             last_rows=fake([R]), free_head_out=fake([1]), admitted=fake([1]))
    a.update(kw)
    return a


def test_batch_build_accepts_and_lists_bindings():
    a = batch_args()
    k = pc.Kernels.PagedBatchBuild(**a)
    assert k.name == "PagedBatchBuild" and k.function_names == ["paged_batch_build"]
    acc = [t[3] for t in k.tensors]
    assert acc == [pc.Access.read] * 4 + [pc.Access.readWrite] + [pc.Access.write] * 7
    # the state of a loop of steps may be kept in place
    pc.Kernels.PagedBatchBuild(**dict(a, seq_lens=a["cached"], free_head_out=a["free_head"]))


@pytest.mark.parametrize("change,code", [
    (dict(cached=fake([4])), E.tensorShapeMismatch),
    (dict(added=fake([5], D.i64)), E.unsupportedDataTypeCombination),
    (dict(block_table=fake([35])), E.tensorInvalidRank),
    (dict(page_size=0), E.tensorShapeMismatch),
    (dict(page_size=-3), E.tensorShapeMismatch),
    (dict(page_size=1 << 31), E.tensorShapeMismatch),
    (dict(query_start=fake([5])), E.tensorShapeMismatch),
    (dict(slots=fake([63])), E.tensorShapeMismatch),
    (dict(last_rows=fake([6])), E.tensorShapeMismatch),
    (dict(free_head=fake([2])), E.tensorShapeMismatch),
    (dict(admitted=fake([1], D.f32)), E.unsupportedDataTypeCombination),
])
def test_batch_build_refusals(change, code):
    refused(code, pc.Kernels.PagedBatchBuild, **batch_args(**change))


def test_batch_build_refuses_overlap_and_too_many_requests():
    a = batch_args()
    refused(E.tensorShapeMismatch, pc.Kernels.PagedBatchBuild, **dict(a, positions=a["slots"]))
    refused(E.tensorShapeMismatch, pc.Kernels.PagedBatchBuild, **dict(a, seq_lens=a["added"]))
    refused(E.tensorShapeMismatch, pc.Kernels.PagedBatchBuild,
            **dict(a, seq_lens=fake([5], ptr=a["cached"].data_ptr + 4)))  # not the whole of it
    R = 16385
    refused(E.tensorShapeMismatch, pc.Kernels.PagedBatchBuild,
            **batch_args(cached=fake([R]), added=fake([R]), block_table=fake([R, 1]), seq_lens=fake([R]),
                         query_start=fake([R + 1]), last_rows=fake([R])))


def scatter_args(**kw):
    T, nq, nkv, hd, P, ps, dt = 6, 4, 2, 64, 9, 16, D.bf16
    a = dict(qkv=fake([T, (nq + 2 * nkv) * hd], dt), slots=fake([T]), q_out=fake([T, nq, hd], dt),
             k_pages=fake([P, nkv, ps, hd], dt), v_pages=fake([P, nkv, ps, hd], dt), cos=fake([T, hd // 2], D.f32),
             sin=fake([T, hd // 2], D.f32), qk_norm=True, q_norm=fake([hd], D.f32), k_norm=fake([hd], D.f32),
             norm_v=True)
    a.update(kw)
    return a


def test_scatter_accepts():
    k = pc.Kernels.PagedQKVScatter(**scatter_args())
    assert k.function_names == ["paged_qkv_scatter_bf16"] and len(k.tensors) == 9
    k = pc.Kernels.PagedQKVScatter(**scatter_args(cos=None, sin=None, qk_norm=False, q_norm=None, k_norm=None))
    assert len(k.tensors) == 5


@pytest.mark.parametrize("change,code", [
    (dict(qkv=fake([6, 511], D.bf16)), E.tensorShapeMismatch),
    (dict(qkv=fake([6, 512], D.f16)), E.unsupportedDataTypeCombination),
    (dict(qkv=fake([6, 512], D.i32)), E.unsupportedDataTypeCombination),
    (dict(q_out=fake([24, 64], D.bf16)), E.tensorInvalidRank),
    (dict(v_pages=fake([9, 2, 8, 64], D.bf16)), E.tensorShapeMismatch),
    (dict(k_pages=fake([9, 2, 16, 32], D.bf16)), E.tensorShapeMismatch),
    (dict(slots=fake([7])), E.tensorShapeMismatch),
    (dict(slots=fake([6], D.i64)), E.unsupportedDataTypeCombination),
    (dict(sin=None), E.tensorShapeMismatch),
    (dict(cos=fake([6, 64], D.f32)), E.tensorShapeMismatch),
    (dict(cos=fake([6, 32], D.bf16)), E.unsupportedDataTypeCombination),
    (dict(q_norm=fake([63], D.f32)), E.tensorShapeMismatch),
    (dict(qk_norm=False), E.tensorShapeMismatch),
])
def test_scatter_refusals(change, code):
    refused(code, pc.Kernels.PagedQKVScatter, **scatter_args(**change))


def test_scatter_refuses_overlap():
    a = scatter_args()
    refused(E.tensorShapeMismatch, pc.Kernels.PagedQKVScatter, **dict(a, v_pages=a["k_pages"]))
    refused(E.tensorShapeMismatch, pc.Kernels.PagedQKVScatter, **dict(a, q_out=fake([6, 4, 64], D.bf16, a["qkv"].data_ptr)))


def attention_args(**kw):
    T, nq, nkv, hd, P, ps, R, W, dt = 6, 4, 2, 128, 9, 16, 3, 5, D.f16
    a = dict(q=fake([T, nq, hd], dt), k_pages=fake([P, nkv, ps, hd], dt), v_pages=fake([P, nkv, ps, hd], dt),
             block_table=fake([R, W]), seq_lens=fake([R]), query_start=fake([R + 1]), into=fake([T, nq, hd], dt),
             scale=0.1)
    a.update(kw)
    return a


def test_attention_accepts():
    k = pc.Kernels.PagedAttention(**attention_args())
    assert k.name == "PagedAttention"
    assert [t[3] for t in k.tensors] == [pc.Access.read] * 6 + [pc.Access.write]
    window = pc.AttentionMask.causal_sliding_window(7)
    pc.Kernels.PagedAttention(**attention_args(mask=window, sinks=4))
    pc.Kernels.PagedAttention(**attention_args(mask=pc.AttentionMask.bidirectional))


@pytest.mark.parametrize("change,code", [
    (dict(q=fake([6, 3, 128], D.f16), into=fake([6, 3, 128], D.f16)), E.tensorShapeMismatch),
    (dict(q=fake([6, 512], D.f16)), E.tensorInvalidRank),
    (dict(into=fake([6, 4, 64], D.f16)), E.tensorShapeMismatch),
    (dict(into=fake([6, 4, 128], D.f32)), E.unsupportedDataTypeCombination),
    (dict(q=fake([6, 4, 128], D.bf16)), E.unsupportedDataTypeCombination),
    (dict(v_pages=fake([8, 2, 16, 128], D.f16)), E.tensorShapeMismatch),
    (dict(block_table=fake([3, 5], D.i64)), E.unsupportedDataTypeCombination),
    (dict(block_table=fake([15])), E.tensorInvalidRank),
    (dict(seq_lens=fake([4])), E.tensorShapeMismatch),
    (dict(query_start=fake([3])), E.tensorShapeMismatch),
    (dict(sinks=4), E.tensorShapeMismatch),
    (dict(sinks=-1), E.tensorShapeMismatch),
    (dict(mask=pc.AttentionMask(1, 0)), E.tensorShapeMismatch),
    (dict(mask=pc.AttentionMask(3)), E.tensorShapeMismatch),
    (dict(q=fake([6, 4, 520], D.f16), into=fake([6, 4, 520], D.f16), k_pages=fake([9, 2, 16, 520], D.f16),
          v_pages=fake([9, 2, 16, 520], D.f16)), E.tensorShapeMismatch),
])
def test_attention_refusals(change, code):
    refused(code, pc.Kernels.PagedAttention, **attention_args(**change))


def test_attention_refuses_overlap():
    a = attention_args()
    refused(E.tensorShapeMismatch, pc.Kernels.PagedAttention, **dict(a, into=a["q"]))


def sample_args(**kw):
    B, V = 5, 1000
    a = dict(logits=fake([B, V], D.bf16), uniform=fake([B], D.f32), tokens=fake([B]), temperature=fake([B], D.f32),
             top_k=fake([B]), top_p=fake([B], D.f32), min_p=fake([B], D.f32))
    a.update(kw)
    return a


def test_sample_accepts():
    k = pc.Kernels.Sample(**sample_args())
    assert k.function_names == ["sample_bf16"] and len(k.tensors) == 7
    k = pc.Kernels.Sample(fake([1000], D.f32), fake([1], D.f32), fake([1]))
    assert k.function_names == ["sample"] and len(k.tensors) == 3


@pytest.mark.parametrize("change,code", [
    (dict(logits=fake([5, 1000], D.i32)), E.unsupportedDataTypeCombination),
    (dict(logits=fake([], D.f32)), E.tensorInvalidRank),
    (dict(logits=fake([5, 0], D.f32)), E.tensorShapeMismatch),
    (dict(tokens=fake([4])), E.tensorShapeMismatch),
    (dict(tokens=fake([5], D.i64)), E.unsupportedDataTypeCombination),
    (dict(uniform=fake([5], D.bf16)), E.unsupportedDataTypeCombination),
    (dict(temperature=fake([1], D.f32)), E.tensorShapeMismatch),
    (dict(top_k=fake([5], D.f32)), E.unsupportedDataTypeCombination),
    (dict(top_p=fake([6], D.f32)), E.tensorShapeMismatch),
    (dict(min_p=fake([5])), E.unsupportedDataTypeCombination),
])
def test_sample_refusals(change, code):
    refused(code, pc.Kernels.Sample, **sample_args(**change))


def test_sample_refuses_overlap():
    a = sample_args()
    refused(E.tensorShapeMismatch, pc.Kernels.Sample, **dict(a, tokens=a["top_k"]))


def test_encoders_share_an_allocator():
    """An allocator's callbacks live as long as it does: a second encoder over it leaves the first's in place."""
    import ctypes
    import gc

    class Fixed(pc.KernelScratchAllocator):
        def borrow(self, length):
            return 4096 + length, False

    pool = Fixed()
    first = pool._c()
    addresses = [ctypes.cast(getattr(first, n), ctypes.c_void_p).value for n in ("borrow", "release")]
    second = pool._c()
    gc.collect()
    assert [ctypes.cast(getattr(second, n), ctypes.c_void_p).value for n in ("borrow", "release")] == addresses
    out, reused = ctypes.c_void_p(), ctypes.c_int()
    for st in (first, second):
        assert st.borrow(None, 64, ctypes.byref(out), ctypes.byref(reused)) == 0 and out.value == 4160


def test_lengths_that_overflow_are_refused():
    refused(E.tensorShapeMismatch, pc.Kernels.Sample, **sample_args(logits=fake([5, (1 << 21) + 1], D.bf16, 1 << 40)))
    a = attention_args()
    ps = a["k_pages"].shape[2]
    W = (1 << 30) // ps
    R = a["block_table"].shape[0]
    pc.Kernels.PagedAttention(**dict(a, block_table=fake([R, W], ptr=1 << 30)))
    refused(E.tensorShapeMismatch, pc.Kernels.PagedAttention, **dict(a, block_table=fake([R, W + 1], ptr=1 << 30)))


@pytest.mark.parametrize("creator,args", [
    (pc.Kernels.PagedBatchBuild, batch_args), (pc.Kernels.PagedQKVScatter, scatter_args),
    (pc.Kernels.PagedAttention, attention_args), (pc.Kernels.Sample, sample_args)])
def test_addresses_are_checked(creator, args):
    """No memory, or an address that is no multiple of the type's size, is refused for every tensor."""
    a = args()
    creator(**a)
    tensors = {n: t for n, t in a.items() if isinstance(t, pc.Tensor)}
    assert len(tensors) >= 5
    for name, t in tensors.items():
        refused(E.tensorShapeMismatch, creator, **dict(a, **{name: fake(t.shape, t.dtype, 0)}))
        refused(E.tensorShapeMismatch, creator, **dict(a, **{name: fake(t.shape, t.dtype, 0x7E0000000001)}))


@pytest.mark.parametrize("shape", [(1 << 40, 1 << 40), (1 << 62, 4)])
def test_sizes_that_overflow_are_refused(shape):
    refused(E.tensorShapeMismatch, pc.Kernels.Sample, **sample_args(logits=fake(shape, D.bf16, 1 << 40)))
    refused(E.tensorShapeMismatch, pc.Kernels.PagedBatchBuild, **batch_args(block_table=fake(shape, D.i32, 1 << 40)))
