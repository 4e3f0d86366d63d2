"""PagedAttention with scores so large that a number next to them is many powers of two away: each row is then the value
of its largest key, whatever the roundings."""
import pytest

from tests.paged_util import HALF, attention_plain
from tests.test_paged_gpu import attention_case, i32

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dt,hd,size", [("f16", 64, 3e3), ("f16", 128, 3e4), ("f16", 256, 1.5e4), ("bf16", 64, 1e5),
                                        ("bf16", 128, 1e9), ("bf16", 256, 1e17), ("f32", 64, 1e9)])
@pytest.mark.parametrize("new,keys", [([1], [3000]), ([1, 200, 1], [700, 900, 5000])])
def test_attention_of_large_scores(dt, hd, size, new, keys):
    """q and k of normal numbers times sqrt(size). A score is a sum of hd products, off by at most hd 2^-24 of the sum of
    their sizes: rows whose first two keys are not further apart than twice that (and 64, for weights) are left out."""
    import popcorn_b200 as pc
    q, k_pages, v_pages, table, start = attention_case(hd, new, keys, 8, 4, hd, 16, dt, q_scale=size ** 0.5)
    k_pages = (k_pages.float() * size ** 0.5).to(k_pages.dtype)
    scale = hd ** -0.5
    out = torch.zeros_like(q)
    enc = pc.KernelCommandEncoder(pc.KernelLibrary(0), scratch=pc.ScratchPool())
    enc.encode(pc.Kernels.PagedAttention(q, k_pages, v_pages, table, i32(keys), i32(start), into=out, scale=scale))
    torch.cuda.synchronize()
    exp, _, _ = attention_plain(q, k_pages, v_pages, table, keys, start, scale, 0, 0, 0)
    clear = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    for r, n in enumerate(keys):
        j = torch.arange(n, device="cuda")
        k = k_pages[table[r].long()[j // 16], :, j % 16].double()
        for t in range(int(start[r]), int(start[r + 1])):
            last = n - int(start[r + 1]) + t + 1
            for h in range(8):
                s = k[:last, h // 2] @ q[t, h].double() * scale
                err = hd * 2.0 ** -24 * (k[:last, h // 2].abs() @ q[t, h].double().abs() * scale).max()
                top = s.topk(min(2, last)).values
                clear[t, h] = last == 1 or top[0] - top[1] > 2 * err + 64
    assert clear.float().mean() > 0.5
    tol = (2 * HALF[dt] * (1 + HALF[dt]) + 2.0 ** -21) * exp.abs()
    assert ((out.double() - exp).abs() <= tol)[clear].all()
    assert pc.device_error_check(0) == 0
