"""More of the product of 8-bit rows and an 8-bit weight: inner sizes of zero."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def Q():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from cssm_amd import sequence
    return sequence


def test_inner_size_of_zero(Q):
    """refused by the entry point as any K it does not take, not by a division"""
    from cssm_amd._lib import CssmError
    a = Q.quantize_rows(torch.empty((4, 0), device="cuda"))
    assert a.values.shape == (4, 0) and a.scales.shape == (4, 0)
    w = Q.Blocks8(torch.empty((8, 0), dtype=torch.float8_e4m3fn, device="cuda"),
                  torch.empty((1, 0), dtype=torch.float8_e8m0fnu, device="cuda"))
    with pytest.raises(CssmError):
        Q.scaled_matmul(a, w)
