"""PagedAttention and PagedStack at the ends of their ranges: many requests, wide groups, scales that are not positive,
steps of more rows and layers."""
import numpy as np
import pytest

from tests.paged_util import attention_plain, attention_tolerance
from tests.test_paged_gpu import CAUSAL, WINDOW, attention_case, check_attention, i32
from tests.test_paged_stack_gpu import HALF, Server, build, plain_logits

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def encoder():
    import popcorn_b200 as pc
    return pc.KernelCommandEncoder(pc.KernelLibrary(0), scratch=pc.ScratchPool())


@pytest.mark.parametrize("dt,hd,R", [("bf16", 64, 417), ("f16", 128, 1000), ("bf16", 256, 833), ("f16", 64, 5000)])
def test_attention_of_many_requests(dt, hd, R):
    """More requests than threads: each sums a run of them. Single tokens, chunks and idle requests mixed."""
    import popcorn_b200 as pc
    rng = np.random.default_rng(R)
    new = np.where(rng.random(R) < 0.8, 1, rng.integers(0, 40, R))
    keys = new + rng.integers(0, 300, R)
    keys[rng.random(R) < 0.02] += 3000
    case = attention_case(R, new.tolist(), keys.tolist(), 4, 2, hd, 16, dt, extra_rows=1)
    check_attention(pc, encoder(), case, keys.tolist(), dt, pc.AttentionMask.causal, CAUSAL, 0, 0)
    check_attention(pc, encoder(), case, keys.tolist(), dt, pc.AttentionMask.causal_sliding_window(90), WINDOW, 90, 2)


@pytest.mark.parametrize("dt,hd", [("bf16", 64), ("f16", 128), ("bf16", 256), ("f32", 64)])
@pytest.mark.parametrize("nq,nkv", [(17, 1), (40, 1), (96, 2), (128, 1), (260, 2)])
def test_attention_of_wide_groups(dt, hd, nq, nkv):
    """Up to 128 query heads to a KV head share a tile of rows (and more take the other kernel)."""
    import popcorn_b200 as pc
    for new, keys in (([1], [700]), ([9, 1, 0, 5], [200, 3000, 4, 5])):
        case = attention_case(nq + hd, new, keys, nq, nkv, hd, 16, dt)
        check_attention(pc, encoder(), case, keys, dt, pc.AttentionMask.causal, CAUSAL, 0, 0)
        check_attention(pc, encoder(), case, keys, dt, pc.AttentionMask.causal_sliding_window(130), WINDOW, 130, 1)


@pytest.mark.parametrize("dt,hd", [("bf16", 64), ("f16", 128), ("f32", 96)])
@pytest.mark.parametrize("scale", [0.0, -0.1, -1.0, 1e-40])
def test_attention_of_other_scales(dt, hd, scale):
    import popcorn_b200 as pc
    new, keys = [1, 30], [300, 200]
    q, k_pages, v_pages, table, start = attention_case(hd, new, keys, 4, 2, hd, 16, dt)
    out = torch.zeros_like(q)
    encoder().encode(pc.Kernels.PagedAttention(q, k_pages, v_pages, table, i32(keys), i32(start), into=out, scale=scale))
    torch.cuda.synchronize()
    exp, mag, _ = attention_plain(q, k_pages, v_pages, table, keys, start, scale, CAUSAL, 0, 0)
    tol = attention_tolerance(exp, mag, q, k_pages, abs(scale), dt, hd)
    assert ((out.double() - exp).abs() <= tol).all()
    assert pc.device_error_check(0) == 0


@pytest.mark.parametrize("dt,hd,tokens,layers", [("bf16", 128, 300, 3), ("f16", 64, 1024, 1), ("bf16", 64, 1, 2)])
def test_paged_stack_of_other_sizes(dt, hd, tokens, layers):
    """Steps of more (and of a single) token rows, other numbers of layers; nothing sets the device's error word."""
    import popcorn_b200 as pc
    from popcorn_b200.decode import LayerShape, PagedStack
    pc.device_error_check(0)
    shape = LayerShape(hidden=256, q_heads=4, kv_heads=2, head_dim=hd, ffn=512, max_ctx=1100, dtype=dt,
                       attn_scale=hd ** -0.5, activation=0)
    st = PagedStack(pc.KernelLibrary(0), shape, layers, 999, 3, tokens, 250, page_size=16, seed=4)
    sv = Server.__new__(Server)
    sv.st, sv.rng = st, np.random.default_rng(tokens)
    sv.fed, sv.ahead = [[] for _ in range(3)], [[] for _ in range(3)]
    sv.pages, sv.cached, sv.head, sv.table = st.free_pages.cpu().numpy(), [0] * 3, 0, st.block_table.cpu().numpy()
    st.top_k.copy_(torch.tensor([0, 5, 50]))

    def run():
        st.encode_step(st.encoder())

    seen = []
    for r, n in enumerate([tokens, tokens // 2 + 1, 1]):
        sv.prompt(r, n)
    first = [tokens, 0, 0]
    second = [0, tokens - 1, 1] if tokens > 1 else [0, 1, 0]
    second[1] = min(second[1], len(sv.ahead[1]))
    for take in (first, second, [1 if tokens > 2 else 0, 1, 0]):
        seen.append(sv.step(run, take))
    assert pc.device_error_check(0) == 0
    full = [plain_logits(st, ids) if ids else None for ids in sv.fed]
    # (as the served runs' bound: 15 roundings a layer and 2)
    for step in seen:
        for r, (at, got) in step.items():
            exp = full[r][at].cpu()
            assert ((got - exp).norm() / exp.norm()).item() <= (15 * layers + 2) * HALF[dt], (r, at)


@pytest.mark.parametrize("dt,hd,page,window", [("bf16", 64, 16, 0), ("f16", 128, 8, 40), ("f32", 48, 5, 0)])
def test_paged_stack_leaves_no_error(dt, hd, page, window):
    """Served steps, waiting requests and two stacks over one scratch buffer leave the device's error word at 0."""
    import popcorn_b200 as pc
    pc.device_error_check(0)
    mask = pc.AttentionMask.causal_sliding_window(window) if window else None
    a, b = build(dt, hd, page, mask, pages=12 * 16 // page), build(dt, hd, page, mask)
    b.scratch = a.scratch
    servers = [Server(a, 1), Server(b, 2)]
    for sv in servers:
        for r, n in enumerate([37, 1, 100, 3]):
            sv.prompt(r, n)

        def run(st=sv.st):
            st.encode_step(st.encoder())

        for take in ([37, 1, 26, 0, 0, 0], [1, 1, 59, 3, 0, 0], [1, 1, 15, 1, 0, 0], [1, 1, 1, 1, 0, 0]):
            sv.step(run, take)
            assert pc.device_error_check(0) == 0
