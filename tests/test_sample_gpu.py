"""Kernels.Sample on the GPU against the plain form in 64 bits."""
import numpy as np
import pytest

from tests.paged_util import sample_plain, torch_dtype

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def pc():
    import popcorn_b200
    return popcorn_b200


@pytest.fixture(scope="module")
def lib(pc):
    return pc.KernelLibrary(0)


def dev(a, dt=torch.float32):
    return torch.tensor(np.asarray(a), dtype=dt, device="cuda")


def draw(pc, lib, logits, u, t=None, k=None, p=None, m=None):
    tokens = torch.full(logits.shape[:-1], -7, dtype=torch.int32, device="cuda")
    opt = lambda a, d=torch.float32: None if a is None else dev(a, d)
    pc.KernelCommandEncoder(lib).encode(pc.Kernels.Sample(logits, dev(u), tokens, temperature=opt(t),
                                                          top_k=opt(k, torch.int32), top_p=opt(p), min_p=opt(m)))
    torch.cuda.synchronize()
    return tokens.cpu().numpy()


def check(pc, lib, logits, u, t=None, k=None, p=None, m=None):
    got = draw(pc, lib, logits, u, t, k, p, m)
    x = logits.double().cpu().numpy()
    for r in range(x.shape[0]):
        exp = sample_plain(x[r], u[r], 1.0 if t is None else t[r], 0 if k is None else k[r], 1.0 if p is None else p[r],
                           0.0 if m is None else m[r])
        assert got[r] == exp, (r, got[r], exp)


def bell(rows, V, dt, seed, sigma=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (sigma * torch.randn(rows, V, generator=g, device="cuda")).to(torch_dtype(dt))


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,V", [(5, 1), (6, 2), (9, 31), (40, 1000), (3, 8193), (2, 50257), (1, 256000), (20, 131072),
                                    (200, 3001)])
def test_sample_filters(pc, lib, dt, rows, V):
    rng = np.random.default_rng(rows + V)
    x = bell(rows, V, dt, rows * V)
    u = rng.random(rows).astype(np.float32)
    t = (0.3 + 1.5 * rng.random(rows)).astype(np.float32)
    t[rng.random(rows) < 0.2] = 0.0
    k = rng.integers(0, min(V, 3000) + 2, rows)
    p = (0.2 + 0.9 * rng.random(rows)).astype(np.float32)
    m = (0.2 * rng.random(rows) ** 3).astype(np.float32)
    check(pc, lib, x, u)
    check(pc, lib, x, u, t=t)
    check(pc, lib, x, u, t=t, k=k)
    check(pc, lib, x, u, t=t, p=p)
    check(pc, lib, x, u, t=t, m=m)
    check(pc, lib, x, u, t=t, k=k, p=p, m=m)
    check(pc, lib, x, u, k=np.full(rows, min(V, 50)), p=np.full(rows, 0.95, np.float32))


@pytest.mark.parametrize("V", [7, 5000, 100001])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_sample_ties(pc, lib, V, dt):
    """Equal logits are ordered by index: cuts of top-k and top-p inside them, whole rows of one value."""
    g = torch.Generator(device="cuda").manual_seed(V)
    few = torch.randint(0, 3, (8, V), generator=g, device="cuda").to(torch_dtype(dt)) * 0.5 - 1
    few[0] = 2.25
    few[1] = -0.0
    few[1, ::2] = 0.0  # -0 and +0 are equal
    u = np.linspace(0, 0.999, 8).astype(np.float32)
    for k in (1, 2, V // 3 + 1, V - 1, V, V + 5):
        check(pc, lib, few, u, k=np.full(8, k))
    for p in (0.0, 1e-6, 0.25, 0.5, 0.77, 0.999, 1.0, 3.0):
        check(pc, lib, few, u, p=np.full(8, p, np.float32))
        check(pc, lib, few, u, k=np.full(8, V // 2 + 1), p=np.full(8, p, np.float32))
    for m in (0.3, 0.99, 1.0, 2.0):
        check(pc, lib, few, u, m=np.full(8, m, np.float32))


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [20, 40000])
def test_sample_masks_and_infinities(pc, lib, dt, V):
    """Masks of -inf and of the type's lowest value, NaN, +inf, rows with nothing left."""
    rows = 12
    x = bell(rows, V, dt, V)
    low = torch.finfo(x.dtype).min
    x[0] = -float("inf")
    x[1] = float("nan")
    x[2, 1:] = -float("inf")
    x[3, ::2] = low
    x[4] = low
    x[4, 5] = 1.0
    x[5] = low  # every token as unlikely as the next
    x[6, 3::4] = float("nan")
    x[7, 2] = float("inf")
    x[7, 9] = float("inf")
    x[8, :-1] = -float("inf")
    x[9, 1::3] = -float("inf")
    x[10, 0] = torch.finfo(x.dtype).max
    u = np.array([0.5, 0.5, 0.9, 0.3, 0.99, 0.7, 0.2, 0.6, 0.0, 0.999, 0.4, 0.1], np.float32)
    t = np.full(rows, 0.9, np.float32)
    for kw in ({}, dict(k=np.full(rows, 9)), dict(p=np.full(rows, 0.8, np.float32)),
               dict(k=np.full(rows, 15), p=np.full(rows, 0.9, np.float32), m=np.full(rows, 0.01, np.float32)),
               dict(t=np.zeros(rows, np.float32))):
        check(pc, lib, x, u, **dict(dict(t=t), **kw))


def test_sample_odd_parameters(pc, lib):
    """Numbers at and outside the ends of their ranges; NaN switches a filter off, a NaN temperature is greedy."""
    rows, V = 16, 5000
    x = bell(rows, V, "f32", 3)
    nan, inf = float("nan"), float("inf")
    greedy = x.argmax(1).cpu().numpy()
    half = np.full(rows, 0.5, np.float32)
    assert np.array_equal(draw(pc, lib, x, half, t=np.full(rows, nan)), greedy)
    assert np.array_equal(draw(pc, lib, x, half, t=np.full(rows, -1.0)), greedy)
    assert np.array_equal(draw(pc, lib, x, half, t=np.full(rows, 1e-30)), greedy)
    assert np.array_equal(draw(pc, lib, x, half, p=np.full(rows, -1.0)), greedy)
    assert np.array_equal(draw(pc, lib, x, half, m=np.full(rows, 5.0)), greedy)
    free = draw(pc, lib, x, half)
    assert np.array_equal(draw(pc, lib, x, half, p=np.full(rows, nan), m=np.full(rows, nan), k=np.full(rows, -4)), free)
    # an infinite temperature draws every finite token alike
    assert np.array_equal(draw(pc, lib, x, half, t=np.full(rows, inf)), np.full(rows, V // 2))
    check(pc, lib, x, half, t=np.full(rows, 3e38, np.float32))
    # numbers outside [0, 1) are brought into it
    first, last = draw(pc, lib, x, np.zeros(rows)), draw(pc, lib, x, np.full(rows, 0.99999994))
    assert np.array_equal(draw(pc, lib, x, np.full(rows, -3.0)), first)
    assert np.array_equal(draw(pc, lib, x, np.full(rows, nan)), first)
    assert np.array_equal(draw(pc, lib, x, np.full(rows, 1.0)), last)
    assert np.array_equal(draw(pc, lib, x, np.full(rows, inf)), last)


def test_sample_long_vocabulary(pc, lib):
    """A row longer than a cluster's shared memory."""
    x = bell(2, 700001, "f32", 11)
    u = np.array([0.3, 0.9], np.float32)
    check(pc, lib, x, u)
    check(pc, lib, x, u, k=[500, 0], p=[0.9, 0.5])


def test_sample_flat_and_narrow(pc, lib):
    """Rows whose tokens nearly all weigh the same, and nearly equal logits around a large value."""
    V = 256000
    x = bell(6, V, "f32", 5, sigma=1e-3)
    x[3:] += 1000.0
    u = np.array([0.1, 0.5, 0.9, 0.2, 0.6, 0.99], np.float32)
    check(pc, lib, x, u, k=[0, 1000, 100000, 0, 1000, 77777], p=np.array([0.9, 0.5, 0.99, 0.3, 1.0, 0.8], np.float32))


def test_sample_share_of_draws(pc, lib):
    """Evenly spaced numbers draw each token in proportion to its weight: counts differ from it by one at most."""
    n = 4000
    w = np.array([5, 1, 0, 3, 7, 4], np.float64)
    with np.errstate(divide="ignore"):
        x = torch.tensor(np.log(w), dtype=torch.float32, device="cuda").repeat(n, 1)
    got = draw(pc, lib, x, (np.arange(n) + 0.5) / n)
    assert (np.abs(np.bincount(got, minlength=6) - n * w / w.sum()) <= 1.001).all()


def test_sample_unaligned_and_captured(pc, lib):
    """Rows at any element offset; a captured draw replayed with other numbers, on a stream of its own."""
    buf = bell(1, 40007, "bf16", 8).view(-1)
    for off in (1, 2, 3, 7):
        x = buf[off:off + 3 * 13331].view(3, 13331)
        check(pc, lib, x, np.array([0.2, 0.5, 0.8], np.float32), k=[40, 0, 7], p=np.array([0.9, 0.7, 1.0], np.float32))
    x = bell(4, 30000, "f16", 2)
    u = torch.zeros(4, device="cuda")
    tokens = torch.zeros(4, dtype=torch.int32, device="cuda")
    p = dev([0.9] * 4)
    kernel = pc.Kernels.Sample(x, u, tokens, top_p=p)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        pc.KernelCommandEncoder(lib, stream=stream).encode(kernel)
    for i in range(4):
        now = np.array([0.1, 0.4, 0.6, 0.9], np.float32) * (1 - 0.2 * i)
        u.copy_(torch.tensor(now))
        graph.replay()
        torch.cuda.synchronize()
        xs = x.double().cpu().numpy()
        assert tokens.cpu().tolist() == [sample_plain(xs[r], now[r], p=0.9) for r in range(4)]


def test_sample_largest_vocabulary(pc, lib):
    """2^21 equal logits: their weights sum to 2^63."""
    V = 1 << 21
    x = torch.full((3, V), -1.5, dtype=torch.bfloat16, device="cuda")
    u = np.array([0.0, 0.5, 0.75], np.float32)
    assert draw(pc, lib, x, u).tolist() == [0, V // 2, V // 4 * 3]
    assert draw(pc, lib, x, u, p=np.full(3, 0.5)).tolist() == [0, V // 4, V // 8 * 3]
    assert draw(pc, lib, x, u, k=np.full(3, V // 2), p=np.full(3, 0.5)).tolist() == [0, V // 8, V // 16 * 3]


@pytest.mark.parametrize("V", [50, 40001])
def test_sample_infinite_logits(pc, lib, V):
    """+inf logits share all the weight, whatever stands beside them."""
    x = bell(5, V, "f32", V)
    x[:, 3::7] = float("inf")
    x[:, 4] = torch.finfo(torch.float32).max
    x[2, 5] = float("nan")
    u = np.array([0.0, 0.3, 0.5, 0.8, 0.9999], np.float32)
    for kw in ({}, dict(k=np.array([1, 2, 5, V // 7 + 3, V - 1])), dict(p=np.array([0.0, 1e-3, 0.5, 0.9, 1.0], np.float32)),
               dict(k=np.full(5, V // 10), p=np.full(5, 0.37, np.float32), m=np.full(5, 1.0, np.float32))):
        check(pc, lib, x, u, t=np.array([0.5, 1.0, 1e-30, 1e30, 2.0], np.float32), **kw)


def test_sample_ranges_at_the_ends_of_f32(pc, lib):
    """Differences that overflow, differences of a few of the smallest numbers, temperatures that go with them."""
    g = torch.Generator(device="cuda").manual_seed(1)
    r = torch.rand(4, 5000, generator=g, device="cuda") * 2 - 1
    u = np.array([0.2, 0.4, 0.6, 0.8], np.float32)
    for size, t in ((3.4e38, 3e38), (3.4e38, float("inf")), (1e-44, 1e-44), (1e-36, 1.0), (1e-30, 1e-30)):
        x = r * size
        for kw in ({}, dict(k=np.array([3, 1000, 4000, 4999])), dict(p=np.array([0.1, 0.5, 0.9, 0.99], np.float32))):
            check(pc, lib, x, u, t=np.full(4, t, np.float32), **kw)
