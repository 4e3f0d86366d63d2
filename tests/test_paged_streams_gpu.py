"""The paged-step kernels on two streams at once, each with scratch memory of its own: the same bits as one after the other,
called directly and replayed from graphs."""
import pytest

from tests.test_paged_gpu import attention_case, i32

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def work(pc, seed, dt, hd):
    """Kernels over tensors of their own, and their outputs."""
    new, keys = [1, 200, 0, 1], [3000 + 100 * seed, 900, 5, 70]
    q, k_pages, v_pages, table, start = attention_case(seed, new, keys, 8, 4, hd, 16, dt)
    q2, k2, v2, _, _ = attention_case(seed + 50, new, keys, 8, 4, hd, 16, dt)
    slots = torch.arange(q.shape[0], device="cuda", dtype=torch.int32) + 32
    qkv = torch.randn(q.shape[0], 16 * hd, device="cuda").to(q.dtype)
    out, out2 = torch.zeros_like(q), torch.zeros_like(q)
    logits = torch.randn(6, 50000, device="cuda")
    u, tokens, p = torch.rand(6, device="cuda"), i32([0] * 6), torch.full((6,), 0.9, device="cuda")
    lens, starts = i32(keys), i32(start)
    K = pc.Kernels
    kernels = [K.PagedAttention(q, k_pages, v_pages, table, lens, starts, into=out, scale=hd ** -0.5),
               K.PagedQKVScatter(qkv, slots, q2, k2, v2),
               K.PagedAttention(q2, k_pages, v_pages, table, lens, starts, into=out2, scale=hd ** -0.5,
                                mask=pc.AttentionMask.causal_sliding_window(400), sinks=2),
               K.Sample(logits, u, tokens, top_p=p)]
    return kernels, [out, out2, tokens, q2]


@pytest.mark.parametrize("hd", [64, 256])
def test_two_streams_at_once(hd):
    import popcorn_b200 as pc
    lib = pc.KernelLibrary(0)
    sides, graphs, scratch = [], [], [pc.FixedScratch(96 << 20) for _ in range(2)]
    for i, dt in enumerate(("bf16", "f16")):
        kernels, outs = work(pc, i + 1, dt, hd)
        stream = torch.cuda.Stream()
        enc = pc.KernelCommandEncoder(lib, stream=stream, scratch=scratch[i])
        torch.cuda.synchronize()
        enc.encode(*kernels)
        torch.cuda.synchronize()
        sides.append((stream, enc, kernels, outs, [t.clone() for t in outs]))
    torch.cuda.synchronize()

    def check():
        torch.cuda.synchronize()
        for _, _, _, outs, first in sides:
            for t, f in zip(outs, first):
                assert torch.equal(t, f)
                t.zero_()
        torch.cuda.synchronize()

    for _ in range(5):
        for _ in range(10):
            for _, enc, kernels, _, _ in sides:
                enc.encode(*kernels)
        check()
    for (stream, _, kernels, _, _), pool in zip(sides, scratch):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            for _ in range(5):
                pc.KernelCommandEncoder(lib, stream=stream, scratch=pool).encode(*kernels)
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(5):
        for (stream, *_), g in zip(sides, graphs):
            with torch.cuda.stream(stream):
                g.replay()
        check()
    assert pc.device_error_check(0) == 0
