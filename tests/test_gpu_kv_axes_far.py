"""Positions of several axes as far out as they may be: floats of magnitudes up to 2^31, negative ones too."""
import numpy as np
import pytest

import gfd_amd
import test_gpu_kv4_append as append
from paged_kv_ref import BF16, E4M3, FP16

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def device():
    assert gfd_amd.device_count() > 0, "no GPU visible to libgfd_amd.so"
    assert gfd_amd.lib().gfd_set_device(0) == 0


@pytest.fixture(autouse=True)
def far(monkeypatch):
    """Step's positions are 0.37 times integers below `far`: from -2^31 to 2^31 / 2 here."""
    init = append.Step.__init__

    def step(self, rng, *args, **kw):
        init(self, rng, *args, **kw)
        low = np.float32(-2.0 ** 31) + self.positions * np.float32(4)
        self.positions[...] = np.where(np.arange(self.positions.shape[1]) % 2, low, self.positions)
        assert np.abs(self.positions).max() <= 2.0 ** 31 and self.positions.min() < -2.0 ** 30
        self.buffers["positions"].upload(np.ascontiguousarray(self.positions).view(np.uint8).reshape(-1))
    monkeypatch.setattr(append.Step, "__init__", step)


def wider(step, x, turned):
    """Of 16- and 8-bit caches the angle, in turns, is off by three roundings of 64 bits: those of 1 / 2 pi, of its product
    with the frequency and of that with the position."""
    y, off = turned(step, x)
    half = len(step.inv_freq)
    angle = np.abs(step.positions[step.axis].T.astype(np.float64) * step.inv_freq.astype(np.float64))[:, None]
    ia, ib = ((np.arange(0, 2 * half, 2), np.arange(1, 2 * half, 2)) if step.pairs else
              (np.arange(half), np.arange(half, 2 * half)))
    off[..., ia] += 3 * 2.0 ** -53 * angle * (np.abs(x[..., ia]) + np.abs(x[..., ib]))
    off[..., ib] = off[..., ia]
    return y, off


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("dtype,cache", [(BF16, 3), (FP16, 3), (BF16, BF16), (FP16, FP16), (BF16, E4M3)])
def test_positions_of_large_magnitude(dtype, cache, pairs, monkeypatch):
    kw = dict(pairs=pairs, axes=3, turns=True, float_positions=True, far=1 << 31)
    if cache == 3:
        append.append4(61, "block", dtype, 128, 128, 40, **kw)
    else:
        turned = append.Step.turned
        monkeypatch.setattr(append.Step, "turned", lambda step, x: wider(step, x, turned))
        append.append16(61, "block", dtype, cache, 128, 128, 40, **kw)
