"""PagedAttention and scratch memory from a caller's own allocator."""
import pytest

from tests.paged_util import attention_plain, attention_tolerance
from tests.test_paged_gpu import attention_case, i32

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_attention_refuses_unaligned_scratch():
    """Pieces of rows go to scratch in 16-byte accesses: memory off a 16-byte border is refused before any launch, and the
    next borrow works."""
    import popcorn_b200 as pc

    class Bump(pc.FixedScratch):
        off = 4

        def borrow(self, length):
            ptr, reused = super().borrow(length + 16)
            return ptr + self.off, reused

        def release(self, ptr):
            super().release(ptr - self.off)

    q, k_pages, v_pages, table, start = attention_case(1, [1, 40], [900, 300], 8, 4, 128, 16, "bf16")
    out = torch.full_like(q, 3.0)
    kernel = pc.Kernels.PagedAttention(q, k_pages, v_pages, table, i32([900, 300]), i32(start), into=out, scale=0.09)
    pool = Bump(64 << 20)
    enc = pc.KernelCommandEncoder(pc.KernelLibrary(0), scratch=pool)
    for off in (4, 8):
        pool.off = off
        with pytest.raises(pc.PopcornError) as e:
            enc.encode(kernel)
        assert e.value.code == pc.PopcornError.tensorAllocationFailed and "16 bytes" in str(e.value)
        torch.cuda.synchronize()
        assert (out == 3.0).all()
    pool.off = 16
    enc.encode(kernel)
    torch.cuda.synchronize()
    exp, mag, _ = attention_plain(q, k_pages, v_pages, table, [900, 300], start, 0.09, 0, 0, 0)
    assert ((out.double() - exp).abs() <= attention_tolerance(exp, mag, q, k_pages, 0.09, "bf16", 128)).all()
