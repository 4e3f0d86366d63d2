"""The paged-step operators in a run, as a server uses them: PagedStack serves
requests whose prompts come whole, in chunks or late, next to others that
decode, and every step's tables, logits and tokens are checked.

Logits are compared, as vectors, with a plain model in 64 bits over the whole
sequence. A 16-bit step rounds about 15 times a layer (norms, q / k / v,
weights and output of the attention, products, activation, sums), each time by
half a step of the type of its own size at most, and random weights keep that
ratio: (15 layers + 2) half steps of the logits' norm bound their error. In
f32 the products' sums dominate: K products sum to within K 2^-24 of their
absolute sum, which is about sqrt(K) of the result's rms; 4 of them a layer and
the head, K at most 512."""
import numpy as np
import pytest

from tests.paged_util import HALF, batch_plain, sample_plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

LAYERS, VOCAB = 2, 999


def plain_logits(st, ids):
    """float64 logits [n, vocab] of one request's tokens."""
    s = st.shape
    n = len(ids)
    x = st.embedding[torch.tensor(ids, device="cuda")].double()
    pos = torch.arange(n, device="cuda", dtype=torch.float64)[:, None]
    cos, sin = [f(pos * st.inv_freq.double())[:, None] for f in (torch.cos, torch.sin)]

    def norm(y, w=None):
        y = y / (y.square().mean(-1, keepdim=True) + s.eps).sqrt()
        return y if w is None else y * (w.double() + 1)

    def rope(y):
        a, b = y.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    i, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")
    seen = j <= i
    if st.mask.kind == 1:
        seen = seen & ((i - j < st.mask.window) | (j < st.sinks))
    for w in st.layers:
        qkv = (norm(x, w.attn_norm) @ w.w_qkv.double().T).view(n, -1, s.Hd)
        q, k, v = qkv.split([s.Nq, s.Nkv, s.Nkv], 1)
        q, k, v = rope(norm(q, w.q_norm)), rope(norm(k, w.k_norm)), norm(v)
        k, v = [t.repeat_interleave(s.Nq // s.Nkv, 1) for t in (k, v)]
        score = torch.einsum("ihd,jhd->hij", q, k) * s.scale
        p = torch.softmax(score.masked_fill(~seen, -float("inf")), -1)
        x = x + torch.einsum("hij,jhd->ihd", p, v).reshape(n, -1) @ w.w_o.double().T
        g, u = (norm(x, w.mlp_norm) @ w.w_gate_up.double().T).chunk(2, -1)
        a = torch.nn.functional.gelu(g, approximate="tanh") if s.activation == 0 else torch.nn.functional.silu(g)
        x = x + (a * u) @ w.w_down.double().T
    return norm(x, st.final_norm) @ st.embedding.double().T


def build(dt, hd=64, page=16, mask=None, sinks=0, requests=6, tokens=64, pages=60):
    import popcorn_b200 as pc
    from popcorn_b200.decode import LayerShape, PagedStack
    shape = LayerShape(hidden=256, q_heads=4, kv_heads=2, head_dim=hd, ffn=512, max_ctx=200, dtype=dt,
                       attn_scale=hd ** -0.5, activation=0)
    return PagedStack(pc.KernelLibrary(0), shape, LAYERS, VOCAB, requests, tokens, pages, page_size=page, seed=3,
                      mask=mask or pc.AttentionMask.causal, sinks=sinks)


class Server:
    """Host side of a run: which request gets which tokens in a step."""

    def __init__(self, st, seed=0):
        self.st, self.rng = st, np.random.default_rng(seed)
        R = st.requests
        self.fed = [[] for _ in range(R)]     # tokens in the cache
        self.ahead = [[] for _ in range(R)]   # prompt tokens to come, or the token drawn last
        self.pages = st.free_pages.cpu().numpy()
        self.cached, self.head, self.table = [0] * R, 0, st.block_table.cpu().numpy()
        st.top_k.copy_(torch.tensor([0, 5, 1, 50, 0, 998][:R]))
        st.top_p.copy_(torch.tensor([1.0, 0.9, 1.0, 0.8, 0.5, 1.0][:R]))
        st.min_p.copy_(torch.tensor([0.0, 0.0, 0.0, 0.01, 0.0, 0.2][:R]))
        st.temperature.copy_(torch.tensor([1.0, 0.7, 1.0, 1.3, 0.9, 0.0][:R]))

    def prompt(self, r, n):
        self.ahead[r] += self.rng.integers(0, VOCAB, n).tolist()

    def step(self, run, take):
        """take[r]: how many of request r's tokens this step gets."""
        st, R = self.st, self.st.requests
        new = [self.ahead[r][:take[r]] for r in range(R)]
        added = [len(t) for t in new]
        ids = sum(new, [])[:st.tokens]
        st.added.copy_(torch.tensor(added, dtype=torch.int32))
        st.ids.copy_(torch.tensor(ids + [0] * (st.tokens - len(ids)), dtype=torch.int32))
        u = self.rng.random(R).astype(np.float32)
        st.uniform.copy_(torch.tensor(u))
        run()
        torch.cuda.synchronize()
        exp = batch_plain(self.cached, added, self.pages, self.head, self.table, st.page_size, st.tokens)
        for name, t in (("seq_lens", st.seq_lens), ("query_start", st.query_start), ("positions", st.positions),
                        ("slots", st.slots), ("last_rows", st.last_rows), ("admitted", st.admitted),
                        ("free_head_out", st.free_head)):
            assert t.cpu().tolist() == list(exp[name]), name
        self.cached, self.head, self.table = exp["seq_lens"], exp["free_head_out"][0], exp["block_table"]
        assert np.array_equal(st.block_table.cpu().numpy(), self.table)
        logits = st.logits.double().cpu()
        drawn = st.next.cpu().tolist()
        par = [t.cpu().tolist() for t in (st.temperature, st.top_k, st.top_p, st.min_p)]
        checked = {}
        for r in range(exp["admitted"][0]):
            if not new[r]:
                continue
            self.fed[r] += new[r]
            del self.ahead[r][:len(new[r])]
            assert drawn[r] == sample_plain(logits[r].numpy(), u[r], *[x[r] for x in par])
            checked[r] = (len(self.fed[r]) - 1, logits[r])
            if not self.ahead[r]:
                self.ahead[r] = [drawn[r]]  # it decodes
        return checked


def tolerance(dt):
    if dt == "f32":
        return (4 * LAYERS + 1) * 512 ** 1.5 * 2.0 ** -24
    return (15 * LAYERS + 2) * HALF[dt]


@pytest.mark.parametrize("dt,hd,page,window,sinks", [
    ("f32", 64, 16, 0, 0), ("f32", 48, 5, 30, 3), ("bf16", 64, 16, 0, 0), ("f16", 128, 8, 0, 0), ("bf16", 256, 64, 0, 0),
    ("f16", 64, 24, 40, 2), ("bf16", 128, 16, 17, 0)])
def test_paged_stack_serves(dt, hd, page, window, sinks):
    import popcorn_b200 as pc
    mask = pc.AttentionMask.causal_sliding_window(window) if window else None
    st = build(dt, hd, page, mask, sinks, pages=60 * 16 // page + 12)
    sv = Server(st, seed=hd)
    seen = []

    def run():
        st.encode_step(st.encoder())

    for r, n in enumerate([37, 1, 100, 3]):
        sv.prompt(r, n)
    seen.append(sv.step(run, [37, 1, 26, 0, 0, 0]))      # a prompt, one token, a chunk; the step is full
    seen.append(sv.step(run, [1, 1, 59, 3, 0, 0]))       # two decode beside a chunk and a new prompt
    sv.prompt(5, 17)
    seen.append(sv.step(run, [1, 1, 15, 1, 0, 17]))      # the prompt's rest; a hole in the batch
    # one captured graph for all the steps to come
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    kept = [t.clone() for t in (st.seq_lens, st.free_head)]
    with torch.cuda.graph(graph, stream=stream):
        st.encode_step(st.encoder(stream))
    assert torch.equal(st.seq_lens, kept[0]) and torch.equal(st.free_head, kept[1])
    sv.prompt(4, 33)
    for i in range(12):
        seen.append(sv.step(graph.replay, [1, 1, 1, 1, 11, 1] if i < 3 else [1, i % 2, 1, 1, 1, i % 3]))
    pc.device_error_check(0)
    full = [plain_logits(st, ids) if ids else None for ids in sv.fed]
    for step in seen:
        for r, (at, got) in step.items():
            exp = full[r][at].cpu()
            err = ((got - exp).norm() / exp.norm()).item()
            assert err <= tolerance(dt), (r, at, err)


def test_paged_stack_waits_for_pages():
    """A request that finds no pages, and those after it, wait: their lengths stay and later steps take them."""
    st = build("bf16", 64, 16, pages=8)
    sv = Server(st)

    def run():
        st.encode_step(st.encoder())

    for r, n in enumerate([40, 50, 60, 5]):
        sv.prompt(r, n)
    assert set(sv.step(run, [20, 30, 14, 0, 0, 0])) == {0, 1, 2}      # 2 + 2 + 1 pages
    # 40, 50, 38 and 5 tokens want 1, 2, 2 and 1 pages more and there are 3: the third waits, and so does the fourth
    assert set(sv.step(run, [20, 20, 24, 5, 0, 0])) == {0, 1}
    assert sv.cached == [40, 50, 14, 0, 0, 0] and sv.head == 8
    # the first request ends: its three pages go back to the list
    st.free_pages[5:] = st.block_table[0, :3]
    st.free_head.fill_(5)
    st.seq_lens[0] = 0
    sv.pages, sv.head, sv.cached[0] = st.free_pages.cpu().numpy(), 5, 0
    assert set(sv.step(run, [0, 1, 24, 5, 0, 0])) == {1, 2, 3}


def test_two_stacks_share_a_stream_and_a_scratch_pool():
    """Two captured stacks with one scratch buffer replay one after the other on a stream: each as if alone."""
    a, b = build("f16", 128, 16), build("f16", 128, 16)
    b.scratch = a.scratch
    stream = torch.cuda.Stream()
    graphs = []
    for st in (a, b):
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=stream):
            st.encode_step(st.encoder(stream))
        graphs.append(g)
    for st in (a, b):
        st.added[0] = 50
        st.ids.copy_(torch.arange(64, dtype=torch.int32) * 7 % VOCAB)
    with torch.cuda.stream(stream):
        for _ in range(3):
            for g in graphs:
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(a.logits, b.logits) and torch.equal(a.seq_lens, b.seq_lens) and a.seq_lens[0] == 150
