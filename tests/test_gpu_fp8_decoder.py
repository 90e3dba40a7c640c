"""The FlashDecoder with block-scaled FP8 linears (DecoderSession, linears =
"fp8_block") against the oracle's decoder whose block linears round both of
their operands to block-scaled FP8 (64-bit definition, oracle/fp8_block.py).

Tolerance. Device and oracle round to E4M3 at the same places, but values that
differ by bf16 rounding (2^-9) before a rounding of step s ~ 2^-3.5 come out a
step apart in a share 2^-9 / s of cases: an rms difference of sqrt(2^-9 s) ~
1.3e-2 of the operand, 12 times bf16's own 1.1e-3. The bf16 decode's bound on
the mean error is 6e-3 (tests/test_gpu_decoder.py), so here 12 x 6e-3 = 0.072
(RGB in [-1, 1]). A wrong weight, bias, norm or order gives errors of the size
of the RGB values themselves, ten times that."""
import numpy as np
import pytest
import torch

from oracle import flashdecoder as ofd
from oracle import fp8_block as o8
from tests.golden import recipes
from tests.test_gpu_decoder import _oracle, _session
from tests.util import assert_no_device_error

pytestmark = pytest.mark.gpu


def _held(x):
    flat = np.asarray(x, np.float64).reshape(-1, x.shape[-1])
    return o8.values(*o8.quantize(flat)).reshape(x.shape).astype(np.float32)


@pytest.mark.parametrize("tag", sorted(recipes.DECODER_CASES))
def test_fp8_decode_stream_matches_oracle(tag, monkeypatch):
    plain = ofd._linear
    weights = {}

    def linear(x, p, name):
        if ".blocks." not in name:
            return plain(x, p, name)
        if name not in weights:
            weights[name] = o8.values(*o8.quantize_weight(np.asarray(p[name + ".weight"], np.float64)))
        y = _held(x) @ weights[name].astype(np.float32).T
        return y + p[name + ".bias"]

    monkeypatch.setattr(ofd, "_linear", linear)
    lat, _, _, lr = recipes.decoder_inputs(tag)
    sess, orc = _session(tag, linears="fp8_block"), _oracle(tag)
    got = [r.float().cpu().numpy()[0] for r in sess.step(torch.from_numpy(lat).cuda(),
                                                          lr_up=torch.from_numpy(lr).cuda())]
    off = 0
    for i, g in enumerate(got):
        take = 1 if i == 0 else 4
        ref, _, _ = orc.step(lat[0, :, i], lr[0, :, off:off + take])
        off += take
        err = np.abs(g - ref).mean()
        assert err <= 0.072, (i, float(err), float(np.abs(ref).mean()))
    assert_no_device_error()


def test_fp8_graph_replay_equals_eager():
    tag = "s"
    c = recipes.DECODER_CASES[tag]
    g = torch.Generator().manual_seed(9)
    lat = torch.randn(1, 48, 6, c["h"], c["w"], generator=g).cuda()
    lr = (torch.rand(1, 3, 21, 16 * c["h"], 16 * c["w"], generator=g) * 2 - 1).cuda()
    eager, graphed = _session(tag, linears="fp8_block"), _session(tag, linears="fp8_block")
    a = [r.clone() for r in eager.step(lat, lr_up=lr)]
    b = [r.clone() for r in graphed.step(lat[:, :, :2], lr_up=lr[:, :, :5])]
    graphed.capture()
    b += [r.clone() for r in graphed.step(lat[:, :, 2:], lr_up=lr[:, :, 5:])]
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_linears_argument():
    with pytest.raises(ValueError, match="fp8_block"):
        _session("s", linears="int8")
