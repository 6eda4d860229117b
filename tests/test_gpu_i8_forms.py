"""Every form that the rules on sizes choose for products and rows in 8 bits: one to four tokens by wide and by long matrices, tiles of every size that go from one to the next, every number of blocks that share a
tile's columns, rows of every width by few and by many."""
import pytest
import torch

from test_gpu_i8 import BF, DEV, check_codes, check_matmul, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 2, 3, 4])
@pytest.mark.parametrize("I", [4112, 5136, 8192, 8208, 12288, 12304, 14336, 16384])
def test_few_tokens_by_wide_matrices(T, I):
    """More than 4096 columns: two to four loads of a row by a warp; few rows, and some by a block."""
    for O in (7, 1000):
        check_matmul(T, O, I)


@pytest.mark.parametrize("T", [1, 2, 3, 4])
@pytest.mark.parametrize("O,I", [(9600, 4096), (9500, 4112), (9500, 5136), (80000, 64), (40000, 1040), (160000, 80)])
def test_few_tokens_by_long_matrices(T, O, I):
    """32 rows of the matrix and more for a warp: eight (of wide rows four) at a time; more rows a block than it sums at once."""
    check_matmul(T, O, I)


@pytest.mark.parametrize("T", [1, 2, 3, 4])
@pytest.mark.parametrize("I", [16, 64, 512, 528, 1536, 2576, 3584, 4096])
def test_few_tokens_by_narrow_matrices(T, I):
    for O in (1, 17, 3001):
        check_matmul(T, O, I)


@pytest.mark.parametrize("T,O,I", [(3, 13000, 8192), (4, 4096, 16400), (2, 300, 16400), (1, 5, 65536), (4, 16500, 4096)])
def test_few_tokens_by_matrices_that_tensor_cores_take(T, O, I):
    check_matmul(T, O, I)


@pytest.mark.parametrize("T,O,I", [(9, 60000, 272), (20, 60000, 272), (32, 39000, 144), (33, 60000, 272), (64, 39000, 1040), (65, 30000, 144), (100, 40000, 272), (128, 19200, 1040), (127, 60001, 16),
                                   (533, 17888, 96), (200, 40000, 128)])
def test_tiles_one_after_the_other(T, O, I):
    """More tiles of 16, 32, 64 and 128 tokens than there are thread blocks."""
    check_matmul(T, O, I)


@pytest.mark.parametrize("shared", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("T", [5, 16, 27, 32, 50, 64])
def test_columns_that_blocks_share(T, shared):
    """One block of 128 columns for each eighth of a tile's tokens is what a thread block of a cluster wants at least."""
    chunks = (2 if T <= 16 else 4 if T <= 32 else 8) * shared
    for O, more in ((128, 0), (130, 48)):
        check_matmul(T, O, 128 * chunks + more)


@pytest.mark.parametrize("T,O,I", [(128, 600, 8192), (300, 129, 4096), (512, 520, 2064)])
def test_columns_of_several_tiles_that_blocks_share(T, O, I):
    check_matmul(T, O, I)


# rows and widths: 64 x 4, 128 x 4, 256 x 2, 256 x 4 threads by groups for many rows; 512 x 1, 2, 4, 8, 16 for few
ROWS = [(300, 8), (300, 2048), (2400, 2056), (2400, 4096), (300, 2056), (300, 4096), (2367, 4088), (300, 4104), (2400, 8192), (5, 4096), (5, 4104), (295, 8200), (2, 16384), (2, 16392), (300, 16392), (2, 32776), (1, 65536)]


@pytest.mark.parametrize("B,n", ROWS)
@pytest.mark.parametrize("residual", [True, False])
def test_norms(B, n, residual):
    g = torch.Generator().manual_seed(B + n)
    a, r = (torch.randn(B, n, generator=g) * 3).to(BF).to(DEV), torch.randn(B, n, generator=g).to(BF).to(DEV)
    w = (1 + 0.3 * torch.randn(n, generator=g)).to(BF).to(DEV)
    h, codes, scales = ops().add_rmsnorm_i8(a, r if residual else None, w, eps=1e-5)
    assert torch.equal(h, (a.float() + r.float()).to(BF) if residual else a)
    # the root, two products, the division, the maximum and 127 / 128 are rounded to 32 bits
    check_codes(codes, scales, h.double() / torch.sqrt(h.double().square().mean(-1, keepdim=True) + 1e-5) * w.double(), 8 * 2.0 ** -24)


@pytest.mark.parametrize("B,n", ROWS)
def test_rows(B, n):
    g = torch.Generator().manual_seed(n)
    x = (torch.randn(B, n, generator=g) * 2.0 ** torch.randint(-9, 9, (B, 1), generator=g).float()).to(BF).to(DEV)
    codes, scales = ops().quantize_rows_i8(x)
    top = x.double().abs().amax(-1, keepdim=True)
    assert torch.equal(codes.double(), torch.round(x.double() * 127 / top))   # values of 16 bits: as exact arithmetic has it
    assert torch.allclose(scales.double(), (top / 127)[:, 0], rtol=2.0 ** -24, atol=0)


@pytest.mark.parametrize("B,n", ROWS)
def test_gated_rows(B, n):
    g = torch.Generator().manual_seed(n + 1)
    x = (torch.randn(B, 2 * n, generator=g) * 4).to(BF).to(DEV)
    codes, scales = ops().quantize_rows_i8(x, gated=True)
    gate, up = x[:, :n].double(), x[:, n:].double()
    # exp to 2 units of its last place, a sum, a quotient, two products: 16 units in all are above it
    check_codes(codes, scales, gate / (1 + torch.exp(-gate)) * up, 16 * 2.0 ** -24)
