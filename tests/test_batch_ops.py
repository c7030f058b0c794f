"""The plain restatement of e4m3 against torch's, on the CPU, and its rounding against the format's definition."""
import numpy as np
import pytest

from batch_ops import E4M3, quantize, to_e4m3, values

torch = pytest.importorskip("torch")


def test_values():
    want = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert ((E4M3 == want) | (np.isnan(E4M3) & np.isnan(want))).all()


def test_rounding():
    rng = np.random.default_rng(0)
    mid = (E4M3[:126] + E4M3[1:127]) / 2
    z = np.concatenate([mid, E4M3[:127], np.nextafter(mid.astype(np.float32), 0), np.nextafter(mid.astype(np.float32), 500),
                        rng.uniform(0, 448, 2000), np.exp(rng.uniform(-12, 6, 2000)), [463.9]]).astype(np.float32)
    z = np.concatenate([z, -z])
    assert (to_e4m3(z) == torch.from_numpy(z).to(torch.float8_e4m3fn).view(torch.uint8).numpy()).all()


def test_blocks():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((130, 272)).astype(np.float32)
    for rows in (1, 128):
        codes, scales = quantize(x, rows)
        v = values(codes, scales, rows)
        assert scales.shape == (-(-130 // rows), 3)
        assert (np.abs(v - x) <= np.maximum(np.abs(x) * 2.0 ** -4, np.repeat(np.repeat(scales, rows, 0)[:130], 128, 1)[:, :272]
                                            * 2.0 ** -10) * 1.0001).all()
