"""gemm_i8 on operands off 16-byte boundaries: every start within 16 bytes, columns that end inside a piece of 16, sums over several
blocks of k, split and not.  The sums are integers below 2^24, so the float result is exact."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def bl(lib):
    if not torch.cuda.is_available():
        pytest.fail("marked gpu but no CUDA device is visible")
    import batchlas_b200
    yield batchlas_b200
    assert batchlas_b200.device_status() == 0


def product(bl, m, n, k, off_a, off_b, lda, ldb, g):
    a = torch.randint(-128, 128, (off_a + m * lda,), generator=g, dtype=torch.int8)
    b = torch.randint(-128, 128, (off_b + n * ldb,), generator=g, dtype=torch.int8)
    # the last column ends with the buffer: nothing behind it may be read
    a, b = a[:off_a + (m - 1) * lda + k].cuda(), b[:off_b + (n - 1) * ldb + k].cuda()
    va, vb = a.as_strided((m, k), (lda, 1), off_a), b.as_strided((n, k), (ldb, 1), off_b)
    c = bl.gemm_i8(va, vb, torch.empty(n, m, device="cuda"))
    assert torch.equal(c.double(), vb.double() @ va.double().T), (m, n, k, off_a, off_b, lda, ldb, bl.last_kernel_name())


@pytest.mark.parametrize("offset", range(16))
def test_every_start(bl, offset):
    g = torch.Generator().manual_seed(offset)
    for n in (5, 20, 70):                                       # the few-column form, tiles split over k, tiles of another width
        product(bl, 140, n, 389, offset, (5 * offset + 3) % 16, 391 + offset, 401, g)
        product(bl, 130, n, 16 + offset, offset, 1, 47, 16 + offset, g)


@pytest.mark.parametrize("m,n,k", [(1500, 1300, 700), (2305, 2100, 129), (257, 130, 1023), (129, 33, 127), (128, 65, 128), (300, 40, 1)])
def test_several_tiles_and_rounds(bl, m, n, k):
    product(bl, m, n, k, 1, 2, k, k + 1, torch.Generator().manual_seed(k))
