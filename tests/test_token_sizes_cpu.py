"""Sizes that do not fit the C entry points' 32-bit arguments are refused before the call, not cut to their lower bits.
Tensors without memory stand for the GPU's."""
import pytest

torch = pytest.importorskip("torch")
from cssm_amd import sequence as Q  # noqa: E402

BF16, F32, F8, E8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.float8_e8m0fnu
WIDE = (1 << 32) + 16


def t(*shape, dtype=F32):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.fixture
def calls(monkeypatch):
    got = []
    monkeypatch.setattr(Q, "_gpu", lambda x, name: 0)
    monkeypatch.setattr(Q, "_call", lambda dev, name, *args: got.append(name))
    return got


def eight(*shape, rows=1):
    m = shape[-2] if rows == 1 else -(-shape[-2] // rows)
    return Q.Blocks8(t(*shape, dtype=F8), t(m, -(-shape[-1] // 128), dtype=E8))


def test_too_wide(calls):
    w = t(WIDE)
    for f in (lambda: Q.rms_norm(t(1, WIDE, dtype=BF16), w),
              lambda: Q.rms_norm_backward(t(1, WIDE, dtype=BF16), None, t(1, WIDE, dtype=BF16), w, 1e-6),
              lambda: Q.quantize_rows(t(2, WIDE, dtype=BF16)),
              lambda: Q.quantize_weight(t(WIDE, 16)),
              lambda: Q.quantize_weight(t(16, WIDE)),
              lambda: Q.scaled_matmul(eight(WIDE, 16), eight(32, 16, rows=128)),
              lambda: Q.scaled_matmul(eight(4, 16), eight(WIDE, 16, rows=128)),
              lambda: Q.scaled_matmul(eight(4, WIDE), eight(32, WIDE, rows=128)),
              lambda: Q.token_scan_step(t(WIDE, 8), t(WIDE, 8), t(8), t(8), t(WIDE, 8)),
              lambda: Q.token_scan_step(t(1, WIDE), t(1, WIDE), w, w, t(1, WIDE)),
              lambda: Q.token_scan(t(1, WIDE, 8), t(1, WIDE, 8), t(8), t(8))):
        with pytest.raises(ValueError, match="2\\^31"):
            f()
    assert not calls


def test_what_fits_is_called(calls):
    w = t(64)
    Q.rms_norm(t(3, 64), w)
    Q.quantize_rows(t(3, 64))
    Q.quantize_weight(t(64, 16))
    Q.scaled_matmul(eight(4, 16), eight(32, 16, rows=128))
    Q.token_scan_step(t(3, 64), t(3, 64), w, w, t(3, 64))
    assert calls == ["cssm_rms_norm", "cssm_quantize_rows", "cssm_quantize_weight", "cssm_scaled_matmul", "cssm_token_scan_step"]
