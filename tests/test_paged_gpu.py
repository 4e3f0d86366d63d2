"""PagedBatchBuild, PagedQKVScatter and PagedAttention on the GPU against
their plain forms in 64 bits (tests/paged_util.py)."""
import numpy as np
import pytest

from tests.paged_util import (HALF, attention_plain, attention_tolerance, batch_plain, scatter_plain, torch_dtype)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def pc():
    import popcorn_b200
    return popcorn_b200


@pytest.fixture(scope="module")
def lib(pc):
    return pc.KernelLibrary(0)


@pytest.fixture()
def enc(pc, lib):
    return pc.KernelCommandEncoder(lib, scratch=pc.ScratchPool())


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


# ---- PagedBatchBuild --------------------------------------------------------

def build(pc, enc, cached, added, free, head, table, page, tokens, in_place=False):
    R = len(cached)
    t = dict(cached=i32(cached), added=i32(added), free_pages=i32(free), free_head=i32([head]), block_table=i32(table),
             seq_lens=i32([7] * R), query_start=i32([7] * (R + 1)), positions=i32([7] * tokens),
             slots=i32([7] * tokens), last_rows=i32([7] * R), free_head_out=i32([7]), admitted=i32([7]))
    if in_place:
        t["seq_lens"], t["free_head_out"] = t["cached"], t["free_head"]
    enc.encode(pc.Kernels.PagedBatchBuild(page_size=page, **t))
    torch.cuda.synchronize()
    return {n: t[n].cpu().numpy() for n in ("seq_lens", "query_start", "positions", "slots", "last_rows",
                                            "free_head_out", "admitted", "block_table")}


def check_build(pc, enc, cached, added, free, head, table, page, tokens):
    exp = batch_plain(cached, added, free, head, table, page, tokens)
    for in_place in (False, True):
        got = build(pc, enc, cached, added, free, head, table, page, tokens, in_place)
        for n, v in exp.items():
            assert np.array_equal(got[n], np.asarray(v, np.int64)), (n, in_place)


@pytest.mark.parametrize("R,page,most,chunk,tokens", [
    (1, 16, 100, 1, 1), (1, 1, 5, 3, 3), (3, 16, 40, 20, 64), (32, 16, 8192, 1, 32), (33, 7, 300, 1, 40),
    (257, 64, 2000, 300, 40000), (1025, 8, 50, 9, 9000), (4099, 3, 20, 4, 12000), (16384, 16, 64, 2, 33000)])
def test_batch_build(pc, enc, R, page, most, chunk, tokens):
    rng = np.random.default_rng(R + page)
    cached = rng.integers(0, most + 1, R)
    added = rng.integers(0, chunk + 1, R)
    cached[rng.random(R) < 0.2] = 0
    need = -(-(cached + added) // page)
    W = int(need.max()) + 1
    ids = rng.permutation(int(need.sum()) + 20)
    table = np.full((R, W), -1)
    at = 0
    for r in range(R):
        n = -(-int(cached[r]) // page)
        table[r, :n] = ids[at:at + n]
        at += n
    check_build(pc, enc, cached, added, ids[at:], 3, table, page, tokens)


def test_batch_build_waits(pc, enc):
    """The first request that does not fit, and all after it, add nothing: tokens, pages, table width."""
    table = np.full((4, 3), -1)
    for tokens, free, added in ((10, 9, [4, 7, 1, 1]), (100, 3, [20, 20, 20, 20]), (100, 9, [5, 49, 1, 0]),
                                (0, 9, [0, 1, 0, 0]), (8, 0, [0, 0, 1, 1]), (100, 9, [2 ** 31 - 1, 1, 1, 1])):
        check_build(pc, enc, [0, 0, 0, 0], added, list(range(50, 50 + free)), 0, table, 16, tokens)


def test_batch_build_odd_inputs(pc, enc):
    """Negative lengths count as none, the head is clamped, page ids of cached keys may be missing (-1)."""
    table = np.array([[5, -1, -1], [-1, -1, -1]])
    check_build(pc, enc, [20, 3], [5, 4], [9, 8, 7], 0, table, 16, 16)  # request 0's second page is missing
    check_build(pc, enc, [-4, 3], [5, -1], [9, 8, 7], -5, table, 16, 16)
    check_build(pc, enc, [0, 0], [5, 4], [9, 8, 7], 99, table, 16, 16)
    check_build(pc, enc, [0, 0], [5, 4], [2 ** 30, 8, 7], 0, table, 16, 16)  # a slot past int32


def test_batch_build_no_requests(pc, enc):
    got = build(pc, enc, [], [], [1, 2], 1, np.zeros((0, 3)), 16, 5)
    assert got["query_start"].tolist() == [0] and got["slots"].tolist() == [-1] * 5
    assert got["free_head_out"].tolist() == [1] and got["admitted"].tolist() == [0]


def test_batch_build_steps_in_a_graph(pc, lib):
    """A captured step, replayed: the state advances in place as the plain form's does."""
    R, page, W, F, T = 3, 4, 8, 24, 8
    stream = torch.cuda.Stream()
    t = dict(cached=i32([0, 5, 2]), added=i32([1, 2, 1]), free_pages=i32(np.arange(100, 100 + F)), free_head=i32([3]),
             block_table=i32([[-1] * W, [1, 2] + [-1] * 6, [3] + [-1] * 7]), query_start=i32([0] * 4),
             positions=i32([0] * T), slots=i32([0] * T), last_rows=i32([0] * R), admitted=i32([0]))
    k = pc.Kernels.PagedBatchBuild(page_size=page, seq_lens=t["cached"], free_head_out=t["free_head"], **t)
    state = [t["cached"].cpu().numpy(), 3, t["block_table"].cpu().numpy()]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        pc.KernelCommandEncoder(lib, stream=stream).encode(k)
    for _ in range(9):
        graph.replay()
        torch.cuda.synchronize()
        exp = batch_plain(state[0], [1, 2, 1], np.arange(100, 100 + F), state[1], state[2], page, T)
        assert t["slots"].cpu().tolist() == exp["slots"]
        assert t["admitted"].cpu().tolist() == exp["admitted"]
        state = [np.array(exp["seq_lens"]), exp["free_head_out"][0], exp["block_table"]]
        assert np.array_equal(t["block_table"].cpu().numpy(), state[2])
        assert t["cached"].cpu().tolist() == exp["seq_lens"] and int(t["free_head"]) == state[1]


# ---- PagedQKVScatter --------------------------------------------------------

@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,nq,nkv,hd,page", [(1, 8, 4, 256, 16), (37, 16, 8, 256, 64), (5, 3, 1, 128, 24),
                                              (19, 12, 4, 64, 8), (33, 4, 2, 96, 7), (3, 2, 1, 6, 1), (70, 5, 5, 512, 3)])
@pytest.mark.parametrize("norm,rope,weights", [(False, False, False), (True, True, True), (False, True, False),
                                               (True, False, False)])
def test_scatter(pc, enc, dt, T, nq, nkv, hd, page, norm, rope, weights):
    g = torch.Generator(device="cuda").manual_seed(T * hd + nq)
    tdt = torch_dtype(dt)
    P = T // page + 3

    def randn(*s):
        return torch.randn(*s, generator=g, device="cuda")

    qkv = (3 * randn(T, (nq + 2 * nkv) * hd)).to(tdt)
    if not norm and not rope:
        qkv[0, :4] = float("nan")  # a copy is a copy of bits
    slots = torch.randperm(P * page, generator=g, device="cuda")[:T].int()
    if T > 2:
        slots[1], slots[T - 1] = -1, P * page  # written nowhere
    k_pages, v_pages = randn(P, nkv, page, hd).to(tdt), randn(P, nkv, page, hd).to(tdt)
    k0, v0 = k_pages.clone(), v_pages.clone()
    q_out = torch.zeros(T, nq, hd, dtype=tdt, device="cuda")
    cos = sin = qn = kn = None
    if rope:
        a = 100 * randn(T, hd // 2)
        cos, sin = a.cos(), a.sin()
    if weights:
        qn, kn = 0.3 * randn(hd), 0.3 * randn(hd)
    norm_v = norm and weights
    enc.encode(pc.Kernels.PagedQKVScatter(qkv, slots, q_out, k_pages, v_pages, cos=cos, sin=sin, qk_norm=norm, q_norm=qn,
                                          k_norm=kn, norm_v=norm_v, eps=1e-6, add_one_to_weight=weights))
    torch.cuda.synchronize()
    q, k, v = scatter_plain(qkv, nq, nkv, hd, cos, sin, norm, qn, kn, norm_v, 1e-6, weights)
    keep = [t for t in range(T) if 0 <= int(slots[t]) < P * page]
    pg, off = slots[keep].long() // page, slots[keep].long() % page
    bits = {"f32": torch.int32, "f16": torch.int16, "bf16": torch.int16}[dt]

    def close(got, exp, raw, exact, pair):
        if exact:
            assert torch.equal(got.contiguous().view(bits), raw.contiguous().view(bits))
            return
        # one rounding at the store; in fp32 the sum of squares (hd terms), the norm and the rotation's two products
        # of values up to `pair` = the larger of |x|, |y| of the rotated pair
        tol = HALF[dt] * exp.abs() + (hd + 16) * 2.0 ** -24 * pair + 1e-30
        assert ((got.double() - exp).abs() <= tol).all()

    def pair(y):
        z = torch.cat([y[..., :hd // 2 or 1].abs() + 0 * y[..., :hd // 2 or 1]] * 2, -1) if hd == 1 else y.abs()
        if hd % 2 == 0:
            a, b = z[..., :hd // 2], z[..., hd // 2:]
            z = torch.cat([a + b, a + b], -1)
        return 2 * z

    raw = qkv.view(T, nq + 2 * nkv, hd)
    plain = not norm and not rope
    close(q_out, q, raw[:, :nq], plain, pair(q))
    close(k_pages[pg, :, off], k[keep], raw[keep][:, nq:nq + nkv], plain, pair(k[keep]))
    close(v_pages[pg, :, off], v[keep], raw[keep][:, nq + nkv:], not norm_v, pair(v[keep]))
    # every other row of the pages is as it was
    for pages, before in ((k_pages, k0), (v_pages, v0)):
        pages[pg, :, off] = before[pg, :, off]
        assert torch.equal(pages.view(bits), before.view(bits))


# ---- PagedAttention ---------------------------------------------------------

def attention_case(seed, new, keys, nq, nkv, hd, page, dt, extra_rows=0, q_scale=1.5):
    """q, pages, table, lengths; every slot that no request holds is NaN or infinite, table entries past a request's
    keys are out of range."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    tdt = torch_dtype(dt)
    counts = [-(-k // page) for k in keys]
    P = sum(counts) + 3
    ids = torch.randperm(P, generator=g, device="cuda")
    table = torch.full((len(keys), max(counts + [1]) + 1), 10 ** 6, dtype=torch.int32, device="cuda")
    start = np.concatenate([[0], np.cumsum(new)])
    T = int(start[-1]) + extra_rows
    k_pages = torch.full((P, nkv, page, hd), float("nan"), dtype=tdt, device="cuda")
    v_pages = torch.full((P, nkv, page, hd), float("inf"), dtype=tdt, device="cuda")
    at = 0
    for r, n in enumerate(keys):
        table[r, :counts[r]] = ids[at:at + counts[r]].int()
        j = torch.arange(n, device="cuda")
        rows = table[r].long()[j // page]
        k_pages[rows, :, j % page] = torch.randn(n, nkv, hd, generator=g, device="cuda").to(tdt)
        v_pages[rows, :, j % page] = torch.randn(n, nkv, hd, generator=g, device="cuda").to(tdt)
        at += counts[r]
    q = (q_scale * torch.randn(T, nq, hd, generator=g, device="cuda")).to(tdt)
    return q, k_pages, v_pages, table, start


def check_attention(pc, enc, case, keys, dt, mask, kind, window, sinks, what=""):
    q, k_pages, v_pages, table, start = case
    hd = q.shape[2]
    scale = hd ** -0.5
    out = torch.full_like(q, 77.0)
    enc.encode(pc.Kernels.PagedAttention(q, k_pages, v_pages, table, i32(keys), i32(start), into=out, scale=scale,
                                         mask=mask, sinks=sinks))
    torch.cuda.synchronize()
    exp, mag, owned = attention_plain(q, k_pages, v_pages, table, keys, start, scale, kind, window, sinks)
    tol = attention_tolerance(exp, mag, q, k_pages, scale, dt, hd)
    got = out.double()
    assert (got[~owned] == 77.0).all(), "rows of no request were written"
    err = (got - exp).abs()[owned]
    bad = ~(err <= tol[owned])
    assert not bad.any(), "%s: %d of %d outside, worst %.3g" % (
        what, int(bad.sum()), bad.numel(), float((err / tol[owned]).nan_to_num(1e9).max()))
    assert pc.device_error_check(0) == 0
    return out


CAUSAL, WINDOW, ALL = 0, 1, 2
SHAPES = [
    # new tokens, keys after them
    ([1], [1]), ([1], [2]), ([1], [129]), ([1], [1000]), ([5], [5]), ([130], [130]), ([17], [300]),
    ([1, 1, 1, 1], [1, 40, 127, 700]), ([3, 1, 64, 0, 129], [3, 513, 64, 9, 400]),
    ([2, 0, 1], [1, 0, 64]),  # a chunk longer than its keys: its first row sees nothing
    ([64] * 9, [64 + 31 * i for i in range(9)]),
]


@pytest.mark.parametrize("dt,nq,nkv,hd,page", [
    ("bf16", 8, 4, 256, 16), ("f16", 8, 4, 256, 64), ("bf16", 16, 2, 128, 32), ("f16", 4, 4, 128, 8),
    ("bf16", 12, 4, 64, 24), ("f16", 8, 1, 64, 128), ("f32", 4, 2, 64, 16), ("bf16", 4, 2, 128, 5),
    ("f16", 6, 3, 80, 16), ("f32", 2, 1, 500, 3), ("bf16", 16, 1, 256, 8), ("f16", 7, 1, 128, 256)])
@pytest.mark.parametrize("kind,window,sinks", [(CAUSAL, 0, 0), (WINDOW, 100, 0), (WINDOW, 70, 4), (WINDOW, 33, 200),
                                               (ALL, 0, 0)])
def test_attention(pc, enc, dt, nq, nkv, hd, page, kind, window, sinks):
    mask = (pc.AttentionMask.causal, pc.AttentionMask.causal_sliding_window(window), pc.AttentionMask.bidirectional)[kind]
    for i, (new, keys) in enumerate(SHAPES):
        case = attention_case(17 * i + hd, new, keys, nq, nkv, hd, page, dt, extra_rows=3)
        check_attention(pc, enc, case, keys, dt, mask, kind, window, sinks, "shape %d" % i)


@pytest.mark.parametrize("dt,hd,page", [("bf16", 256, 16), ("f16", 128, 64), ("bf16", 64, 32)])
def test_attention_long_contexts(pc, enc, dt, hd, page):
    """Single tokens over long contexts (work split over the keys and joined) beside a long chunk."""
    for new, keys in (([1], [20011]), ([1, 1], [9001, 33]), ([300, 1], [5000, 7000]), ([1025], [1500])):
        case = attention_case(len(keys) + hd, new, keys, 8, 4, hd, page, dt)
        check_attention(pc, enc, case, keys, dt, pc.AttentionMask.causal, CAUSAL, 0, 0)
        check_attention(pc, enc, case, keys, dt, pc.AttentionMask.causal_sliding_window(1000), WINDOW, 1000, 64)


@pytest.mark.parametrize("dt,hd,page", [("bf16", 256, 64), ("f16", 128, 16), ("bf16", 64, 8)])
@pytest.mark.parametrize("new,keys", [
    ([700, 1, 1, 130, 0, 1, 1], [6000, 9000, 12000, 3001, 77, 500, 1]),  # chunks and single tokens
    ([1] * 40, [1900 + 13 * i for i in range(40)]),                      # single tokens alone
    ([257] * 23, [257 + 40 * i for i in range(23)]),                     # many short items
])
def test_attention_long_runs(pc, enc, dt, hd, page, new, keys):
    """Steps with more than 16 tiles of 128 keys for each SM: items then count for more than their tiles."""
    nq, nkv = 8, 4
    tokens = 128 // (nq // nkv)  # of an item
    tiles = sum(nkv * -(-(k - n + min(t + tokens, n)) // 128) for n, k in zip(new, keys) for t in range(0, n, tokens))
    assert tiles > 16 * torch.cuda.get_device_properties(0).multi_processor_count
    case = attention_case(hd + len(new), new, keys, nq, nkv, hd, page, dt)
    check_attention(pc, enc, case, keys, dt, pc.AttentionMask.causal, CAUSAL, 0, 0)
    check_attention(pc, enc, case, keys, dt, pc.AttentionMask.causal_sliding_window(3000), WINDOW, 3000, 10)


@pytest.mark.parametrize("dt,hd,page", [("bf16", 256, 16), ("f16", 128, 64), ("bf16", 64, 32), ("f32", 64, 16)])
def test_attention_masked_poison(pc, enc, dt, hd, page):
    """NaN and infinities in keys and values reach the rows that see them, and no other."""
    new, keys = [200, 1, 40], [250, 90, 40]
    case = attention_case(5, new, keys, 4, 2, hd, page, dt)
    q, k_pages, v_pages, table, start = case

    def at(r, j):
        return int(table[r, j // page]), slice(None), j % page

    v_pages[at(0, 240)] = float("nan")      # seen by the last ten rows of request 0 alone
    v_pages[at(0, 3)][:, 5] = float("inf")  # out of the window of the late rows, not of the first
    k_pages[at(2, 39)] = float("nan")       # seen by the last row of request 2 alone
    window = 150
    out = torch.zeros_like(q)
    enc.encode(pc.Kernels.PagedAttention(q, k_pages, v_pages, table, i32(keys), i32(start), into=out, scale=hd ** -0.5,
                                         mask=pc.AttentionMask.causal_sliding_window(window)))
    torch.cuda.synchronize()
    finite = torch.isfinite(out).view(out.shape[0], -1)
    pos = torch.arange(50, 250, device="cuda")
    sees_nan, sees_inf = pos >= 240, (pos - 3 < window)
    assert torch.isnan(out[:200][sees_nan]).all()
    only_inf = sees_inf & ~sees_nan
    assert (out[:200][only_inf][:, :, 5] == float("inf")).all()
    rest = torch.ones(hd, dtype=torch.bool, device="cuda")
    rest[5] = False
    assert torch.isfinite(out[:200][only_inf][:, :, rest]).all()
    assert finite[:200][~sees_inf & ~sees_nan].all()
    assert finite[200:240].all() and torch.isnan(out[240]).all()
    # the untouched rows equal those of a clean cache
    exp, mag, _ = attention_plain(q, k_pages, v_pages, table, keys, start, hd ** -0.5, WINDOW, window, 0)
    tol = attention_tolerance(exp, mag, q, k_pages, hd ** -0.5, dt, hd)
    good = torch.isfinite(exp)
    assert good.any() and ((out.double() - exp).abs() <= tol)[good].all()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_attention_bad_lengths_and_pages(pc, enc, dt):
    """Lengths outside the tensors are clamped, a page id outside the pages sets its bit; other requests are right."""
    new, keys = [4, 1, 3], [40, 100, 30]
    case = attention_case(9, new, keys, 4, 2, 128, 16, dt)
    q, k_pages, v_pages, table, start = case
    good = check_attention(pc, enc, case, keys, dt, pc.AttentionMask.causal, CAUSAL, 0, 0)
    for bad in (-1, k_pages.shape[0], 2 ** 31 - 1, -2 ** 31):
        broken = table.clone()
        broken[1, 2] = bad
        out = torch.zeros_like(q)
        enc.encode(pc.Kernels.PagedAttention(q, k_pages, v_pages, broken, i32(keys), i32(start), into=out,
                                             scale=128 ** -0.5))
        torch.cuda.synchronize()
        assert pc.device_error_check(0) == 32
        assert torch.equal(out[:4], good[:4]) and torch.equal(out[5:], good[5:])
    # lengths and starts out of range: nothing outside the tensors is read or written
    out = torch.zeros_like(q)
    for lens, st in (([-5, 2 ** 31 - 1, 30], start), (keys, [0, 4, 99, 8]), (keys, [-3, 4, 2, 2 ** 30])):
        fixed = table.clone()
        fixed[fixed == 10 ** 6] = 0
        enc.encode(pc.Kernels.PagedAttention(q, k_pages, v_pages, fixed, i32(lens), i32(st), into=out, scale=0.1))
    torch.cuda.synchronize()
    assert pc.device_error_check(0) == 0


def test_attention_empty(pc, enc):
    """No requests, no tokens: nothing is written."""
    q, k_pages, v_pages, table, start = attention_case(1, [2], [5], 4, 2, 128, 16, "bf16")
    out = torch.full_like(q, 3.0)
    enc.encode(pc.Kernels.PagedAttention(q, k_pages, v_pages, table[:0], i32([]), i32([0]), into=out, scale=0.1))
    enc.encode(pc.Kernels.PagedAttention(q[:0], k_pages, v_pages, table, i32([5]), i32([0, 0]), into=out[:0], scale=0.1))
    enc.encode(pc.Kernels.PagedAttention(q, k_pages, v_pages, table, i32([5]), i32([0, 0]), into=out, scale=0.1))
    torch.cuda.synchronize()
    assert (out == 3.0).all()


@pytest.mark.parametrize("dt,hd", [("bf16", 256), ("f16", 128)])
def test_attention_is_repeatable_and_captures(pc, lib, dt, hd):
    """The same bits every time, eagerly and from a graph replayed with other lengths; two graphs over one scratch
    pool on one stream."""
    keys, new = [3000, 700, 129], [1, 30, 129]
    q, k_pages, v_pages, table, start = attention_case(3, new, keys, 8, 2, hd, 32, dt)
    lens, qs = i32(keys), i32(start)
    out = torch.zeros_like(q)
    stream = torch.cuda.Stream()
    pool = pc.FixedScratch(64 << 20)
    kernel = pc.Kernels.PagedAttention(q, k_pages, v_pages, table, lens, qs, into=out, scale=hd ** -0.5)
    eager = pc.KernelCommandEncoder(lib, stream=stream, scratch=pool)
    torch.cuda.synchronize()
    eager.encode(kernel)
    torch.cuda.synchronize()
    first = out.clone()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            pc.KernelCommandEncoder(lib, stream=stream, scratch=pool).encode(kernel)
        graphs.append(graph)
    for graph in graphs * 3:
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
    other = [2990, 31, 400]
    lens.copy_(i32(other))
    for r in range(3):  # the third request now holds more keys than its pages: give it the first's
        table[r] = torch.where(table[r] >= k_pages.shape[0], table[0][:table.shape[1]], table[r])
    graphs[0].replay()
    torch.cuda.synchronize()
    exp, mag, _ = attention_plain(q, k_pages, v_pages, table, other, start, hd ** -0.5, CAUSAL, 0, 0)
    tol = attention_tolerance(exp, mag, q, k_pages, hd ** -0.5, dt, hd)
    good = torch.isfinite(exp)
    assert ((out.double() - exp).abs() <= tol)[good].all()


@pytest.mark.parametrize("n", [1, 40])
def test_attention_far_pages(pc, enc, n):
    """Pages whose byte offset passes 32 bits."""
    hd, page, nkv = 128, 64, 2
    P = (5 << 30) // (nkv * page * hd * 2)
    k_pages = torch.empty(P, nkv, page, hd, dtype=torch.bfloat16, device="cuda")
    v_pages = torch.empty_like(k_pages)
    keys, count = 500, 8
    table = torch.arange(P - count, P, device="cuda", dtype=torch.int32).view(1, count)
    g = torch.Generator(device="cuda").manual_seed(2)
    k_pages[P - count:] = torch.randn(count, nkv, page, hd, generator=g, device="cuda").bfloat16()
    v_pages[P - count:] = torch.randn(count, nkv, page, hd, generator=g, device="cuda").bfloat16()
    q = torch.randn(n, 4, hd, generator=g, device="cuda").bfloat16()
    out = torch.zeros_like(q)
    enc.encode(pc.Kernels.PagedAttention(q, k_pages, v_pages, table, i32([keys]), i32([0, n]), into=out, scale=0.09))
    torch.cuda.synchronize()
    exp, mag, _ = attention_plain(q, k_pages, v_pages, table, [keys], [0, n], 0.09, CAUSAL, 0, 0)
    tol = attention_tolerance(exp, mag, q, k_pages[P - count:], 0.09, "bf16", hd)
    assert ((out.double() - exp).abs() <= tol).all()
