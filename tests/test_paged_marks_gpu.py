"""PagedAttention counts every key exactly once: with q = 0 all visible keys weigh the same, and a value that is zero but
for one key in each column tells whether a row's sum holds that key, and how often. (A tolerance on random values cannot:
over 20000 keys a tile of 128 more or less stays within the roundings of bf16.)"""
import numpy as np
import pytest

from tests.paged_util import HALF, torch_dtype
from tests.test_paged_gpu import ALL, CAUSAL, WINDOW, i32

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

MARK = 4096.0
STEPS = {
    "one": ([1], [20011]),                                                    # cut into pieces all over the GPU
    "chunk and one": ([300, 1], [5000, 7000]),
    "mixed": ([700, 1, 1, 130, 0, 1, 1], [6000, 9000, 12000, 3001, 77, 500, 1]),  # runs of more than 16 tiles a CTA
    "decoding": ([1] * 40, [1900 + 13 * i for i in range(40)]),
    "short": ([257] * 9, [257 + 40 * i for i in range(9)]),
}


@pytest.mark.parametrize("step", list(STEPS))
@pytest.mark.parametrize("dt,nq,nkv,hd,page", [("bf16", 8, 4, 64, 16), ("f16", 8, 4, 64, 24), ("bf16", 16, 2, 128, 64),
                                               ("f16", 8, 4, 128, 8), ("bf16", 8, 4, 256, 16), ("f16", 4, 4, 256, 128)])
def test_attention_counts_each_key_once(step, dt, nq, nkv, hd, page):
    import popcorn_b200 as pc
    new, keys = STEPS[step]
    tdt = torch_dtype(dt)
    rng = np.random.default_rng(hd + page)
    counts = [-(-n // page) for n in keys]
    P = sum(counts) + 1
    ids = torch.from_numpy(rng.permutation(P)).cuda()
    table = torch.full((len(keys), max(counts)), 10 ** 6, dtype=torch.int32, device="cuda")
    k_pages = torch.randn(P, nkv, page, hd, device="cuda").to(tdt)
    v_pages = torch.zeros(P, nkv, page, hd, dtype=tdt, device="cuda")
    start = np.concatenate([[0], np.cumsum(new)])
    marks, at = [], 0  # [nkv * hd] of each request
    for r, n in enumerate(keys):
        table[r, :counts[r]] = ids[at:at + counts[r]].int()
        at += counts[r]
        # borders of tiles, their halves, pages, the windows of the first and last rows, sinks; the rest anywhere
        edges = {0, 1, 2, 3, 9, 10, 63, 64, n - 1, n - 2, n - new[r], n - new[r] - 1, n - new[r] + 1}
        for w in (3000, 200):
            edges |= {n - w, n - w - 1, n - w + 1, n - new[r] - w, n - new[r] - w + 1, n - new[r] - w - 1}
        tiles = rng.integers(0, n // 128 + 1, 30) * 128
        edges |= {int(x) + d for x in tiles for d in (-1, 0, 63, 64)}
        edges = rng.permutation(sorted({e for e in edges if 0 <= e < n}))[:nkv * hd // 2]
        mark = np.concatenate([edges, rng.integers(0, n, nkv * hd - len(edges))])
        marks.append(torch.from_numpy(rng.permutation(mark)).cuda())
        head = torch.arange(nkv * hd, device="cuda") // hd
        column = torch.arange(nkv * hd, device="cuda") % hd
        v_pages[table[r].long()[marks[r] // page], head, marks[r] % page, column] = MARK
    q = torch.zeros(int(start[-1]), nq, hd, dtype=tdt, device="cuda")
    enc = pc.KernelCommandEncoder(pc.KernelLibrary(0), scratch=pc.ScratchPool())
    lens, starts = i32(keys), i32(start)
    for kind, window, sinks in ((CAUSAL, 0, 0), (WINDOW, 3000, 10), (WINDOW, 200, 0), (ALL, 0, 0)):
        mask = (pc.AttentionMask.causal, pc.AttentionMask.causal_sliding_window(max(window, 1)), pc.AttentionMask.bidirectional)[kind]
        out = torch.full_like(q, 77.0)
        enc.encode(pc.Kernels.PagedAttention(q, k_pages, v_pages, table, lens, starts, into=out, scale=hd ** -0.5, mask=mask,
                                             sinks=sinks))
        torch.cuda.synchronize()
        for r, n in enumerate(keys):
            if not new[r]:
                continue
            pos = torch.arange(n - new[r], n, device="cuda")[:, None]

            def sees(j):
                if kind == ALL:
                    return torch.ones(len(pos), len(j), dtype=torch.bool, device="cuda")
                s = j <= pos
                return s & ((pos - j < window) | (j < sinks)) if kind == WINDOW else s

            total = sees(torch.arange(n, device="cuda")).sum(1, keepdim=True)
            exp = (MARK * sees(marks[r]).double() / total).view(len(pos), nkv, 1, hd)
            got = out[int(start[r]):int(start[r + 1])].double().view(len(pos), nkv, nq // nkv, hd)
            # the sums are exact (powers of two, fewer than 2^24 of them); 1 / l, its product and the pieces' weights round in
            # fp32, the store once in the type
            tol = (HALF[dt] + 2.0 ** -20) * exp
            bad = (got - exp).abs() > tol
            assert not bad.any(), (kind, r, bad.nonzero()[:4].tolist())
    assert pc.device_error_check(0) == 0
