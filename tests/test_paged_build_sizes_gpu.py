"""PagedBatchBuild at the sizes where its launch changes: one CTA or eight, one token row a thread or four."""
import numpy as np
import pytest

from tests.test_paged_gpu import check_build, enc, lib, pc  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("tokens", [31, 1023, 1024, 1025, 1027, 4095, 4096, 4097, 8191, 8192, 8193, 8195])
@pytest.mark.parametrize("chunk,page", [(1, 16), (3, 1), (600, 16)])
def test_batch_build_sizes(pc, enc, tokens, chunk, page):  # noqa: F811
    """Steps that fill their token rows, leave some, or have too many tokens, so that the last requests wait."""
    rng = np.random.default_rng(tokens + chunk)
    for share in (1.0, 0.7, 1.2):
        added = []
        while sum(added) < int(tokens * share):
            added.append(int(rng.integers(0 if chunk > 1 else 1, chunk + 1)))
        if share == 1.0:
            added[-1] -= sum(added) - tokens
        added = np.array(added)
        R = len(added)
        cached = rng.integers(0, 50, R)
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
