"""PagedAttention where small weights matter: one key that outweighs every
other by far, with a value of zero, so that the output is the sum of many
small weights' values."""
import pytest

from tests.paged_util import attention_plain, attention_tolerance
from tests.test_paged_gpu import i32, torch_dtype

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

KEYS = 40000


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 64), (256, 32)])
@pytest.mark.parametrize("at", [0, 7, 20001, KEYS - 1])
def test_attention_sums_small_weights(dt, hd, page, at):
    """Key `at` has the score 17.4, all others 0: each of them weighs exp(-17.4) = 2^-25.1 of it, all together 1.1e-3.
    40 requests share the pages, so that the pieces are long. The bound is the other tests': weights to half a step of
    the type each, relative to themselves."""
    import popcorn_b200 as pc
    nq, nkv, R = 8, 4, 40
    g = torch.Generator(device="cuda").manual_seed(hd + at)
    tdt = torch_dtype(dt)
    P = KEYS // page
    scale = hd ** -0.5
    k_pages = torch.zeros(P, nkv, page, hd, dtype=tdt, device="cuda")
    v_pages = (0.5 + torch.rand(P, nkv, page, hd, generator=g, device="cuda")).to(tdt)
    table = torch.randperm(P, generator=g, device="cuda").int().view(1, P)
    row = int(table[0, at // page])
    k_pages[row, :, at % page, 0] = 4.0
    v_pages[row, :, at % page] = 0.0
    q = torch.zeros(1, nq, hd, dtype=tdt, device="cuda")
    q[..., 0] = 17.4 / 4.0 / scale
    out = torch.zeros(R, nq, hd, dtype=tdt, device="cuda")
    enc = pc.KernelCommandEncoder(pc.KernelLibrary(0), scratch=pc.ScratchPool())
    enc.encode(pc.Kernels.PagedAttention(q.repeat(R, 1, 1), k_pages, v_pages, table.repeat(R, 1), i32([KEYS] * R),
                                         i32(range(R + 1)), into=out, scale=scale))
    torch.cuda.synchronize()
    exp, mag, _ = attention_plain(q, k_pages, v_pages, table, [KEYS], [0, 1], scale, 0, 0, 0)
    assert exp.min() > 2.0 ** -14  # (normal numbers in every type)
    tol = attention_tolerance(exp, mag, q, k_pages, scale, dt, hd)
    err = ((out.double() - exp).abs() / tol).max().item()
    assert err <= 1.0, err
    assert pc.device_error_check(0) == 0
