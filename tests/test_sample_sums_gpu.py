"""Sample at the largest vocabulary: its sums of weights are exact there too."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_sample_sums_are_exact_at_the_largest_vocabulary():
    """Weights of 2^42 - k: l = -k 2^-42 below a largest logit of 0. Each half of the row sums to A = 2^62 - 768, so with
    u = 1/2 the goal is A, the first half does not exceed it, and the token is the first of the second half. A is a tie
    of 512ths on the way to a double: a sum of the first half that is off by one upwards, and one of the second half by
    one downwards, leave the goal as it is and put its place into the first half, where no token exceeds it. Such sums
    come about where one thread adds more than 2^11 weights in a double (tokens 1, 7 .. 10, 135 .. 138, ... of a
    65536-token segment of a row that starts 4 bytes after a 16-byte border, with so many rows that each has one CTA): an odd sum above 2^53
    is rounded to a multiple of 4, so k = 1 in one such share and k = 3 in another give +1 and -1."""
    import popcorn_b200 as pc
    V, rows = 1 << 21, 80
    k = np.zeros(V, np.int64)
    k[15 * 65536 + 7], k[23] = 1, 767        # first half: a share of 2049 tokens; one of 2048
    k[20 * 65536 + 7], k[V // 2 + 23] = 3, 765
    weights = (1 << 42) - k
    cum = np.cumsum(weights.astype(np.uint64))
    assert int(cum[V // 2 - 1]) == (1 << 62) - 768 and int(cum[-1]) == (1 << 63) - 1536
    row = torch.tensor(k, device="cuda").double().mul(-2.0 ** -42).float()
    store = torch.empty(rows * V + 1, device="cuda")
    x = store[1:].view(rows, V)
    x[:] = row
    u = np.full(rows, 0.5, np.float32)
    u[1], u[2] = 0.25, 0.0
    exp = [V // 2, V // 4, 0] + [V // 2] * (rows - 3)
    for r in range(3):  # in integers: the first index whose sum exceeds u times the total (u in 4ths)
        goal = int(u[r] * 4) * int(cum[-1])
        assert goal < 4 * int(cum[exp[r]]) and (exp[r] == 0 or 4 * int(cum[exp[r] - 1]) <= goal)
    tokens = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    pc.KernelCommandEncoder(pc.KernelLibrary(0)).encode(pc.Kernels.Sample(x, torch.tensor(u, device="cuda"), tokens))
    torch.cuda.synchronize()
    assert tokens.cpu().tolist() == exp
