"""Every launch of the FlashDecoder's block-scaled FP8 blocks (DecoderSession,
linears="fp8_block") against the reference's state dict.

An error bound on the decoded RGB cannot tell this path from its faults: E4M3
roundings that fall differently move the RGB by as much as a lost bias does. So
the session's buffers are copied after each launch of one step, and each launch
is checked from the buffers before it: its own inputs as the device had them,
the layer's parameters straight from the state dict, held in 8 bits by the
64-bit definition (oracle/fp8_block.py). The bounds are those of the operators
(tests/test_gpu_fp8_block.py): quantizers and stored sums exact, norms and gated
products within a code's rounding, products between the roundings of the lowest
and the highest sum. Each check is also given the parameters with a fault
planted and has to refuse them."""
import numpy as np
import pytest
import torch

from oracle import fp8_block as o8
from tests.golden import recipes
from tests.test_gpu_decoder import _session
from tests.test_gpu_fp8_block import DELTA, assert_held_near, assert_rounded_from, sum_slack
from tests.util import assert_no_device_error

pytestmark = pytest.mark.gpu

BUFFERS = ("rows8", "rows8_s", "act8", "act8_s", "delta", "qkv", "att", "x", "hr")
BLOCK = ["rc_fp8_block_rms_norm", "rc_fp8_block_gemm", "rc_fd_kv_norm", "rc_fd_rope_gather",
         "rc_local_gqa_attention", "rc_fp8_block_quantize", "rc_fp8_block_gemm", "rc_fp8_block_rms_norm",
         "rc_fp8_block_swiglu_gemm", "rc_fp8_block_gemm"]


def _recorded(tag, monkeypatch):
    """(session, [(entry point, buffers after it)]) of the second step: no empty cache, both stacks."""
    from recavsr_b200 import _lib
    sess = _session(tag, linears="fp8_block")
    lat, _, _, lr = (None if a is None else torch.from_numpy(a).cuda() for a in recipes.decoder_inputs(tag))
    list(sess.step(lat[:, :, :1], lr_up=lr[:, :, :1]))
    log, call = [], _lib.call

    def recording(name, *args):
        call(name, *args)
        log.append((name, {b: getattr(sess, b).clone() for b in BUFFERS}))

    with monkeypatch.context() as patch:
        patch.setattr(_lib, "call", recording)
        list(sess.step(lat[:, :, 1:2], lr_up=lr[:, :, 1:5]))
    assert_no_device_error()
    return sess, log


def _blocks(sess, log):
    """(prefix, stream buffer, tokens, first of its stack, last, [buffers before and after each launch]) of each block."""
    from_start = [i for i, (name, _) in enumerate(log) if name == BLOCK[0]][::2]
    stacks = [("backbone", "x", sess.n, len(sess.backbone.layers)),
              ("temporal_refinement", "hr", 4 * sess.n, len(sess.refinement.layers))]
    assert len(from_start) == sum(s[3] for s in stacks)
    at = iter(from_start)
    for name, stream, tokens, depth in stacks:
        for layer in range(depth):
            i = next(at)
            assert [n for n, _ in log[i:i + len(BLOCK)]] == BLOCK
            yield (f"{name}.blocks.{layer}.", stream, tokens, layer == 0, layer + 1 == depth,
                   [b for _, b in log[i - 1:i + len(BLOCK)]])


def _f64(t):
    return t.double().cpu().numpy()


def _operand(buffers, name, tokens, cols):
    from recavsr_b200.runtime import fp8_block
    codes, scales = buffers[name][:tokens], buffers[name + "_s"][:fp8_block.scale_numel(tokens, cols)]
    return codes, scales, fp8_block.dequantize(codes, scales).double()


def _weight(p, names):
    w = np.concatenate([np.asarray(p[n + ".weight"], np.float64) for n in names])
    return torch.from_numpy(o8.values(*o8.quantize_weight(w))).cuda()


def _bias(p, names):
    return torch.from_numpy(np.concatenate([np.asarray(p[n + ".bias"], np.float64) for n in names])).cuda()


def check_product(p, names, operand, out, residual=None):
    _, _, av = operand
    w, b = _weight(p, names), _bias(p, names)
    ref, slack = av @ w.t() + b, sum_slack(av, w, w.shape[1])
    slack = slack + 2.0 ** -23 * (b.abs() + ref.abs())
    if residual is not None:
        ref = ref + residual.double()
        slack = slack + 2.0 ** -23 * (residual.double().abs() + ref.abs())
    assert_rounded_from(out, ref, slack)


def check_norm(p, name, eps, x, delta, stored, codes, scales):
    y, h = o8.rms_norm(_f64(x), np.asarray(p[name + ".weight"], np.float64), eps, None if delta is None else _f64(delta))
    assert_held_near(codes, scales, y, np.abs(y) * DELTA)
    # the sum of two bf16 values rounded to fp32 and then to bf16
    assert torch.equal(stored, x if delta is None else (x.float() + delta.float()).bfloat16())


def check_gated(p, f, operand, codes, scales):
    _, _, av = operand
    wg, wu = _weight(p, [f + "gate"]), _weight(p, [f + "up"])
    g, u = av @ wg.t() + _bias(p, [f + "gate"]), av @ wu.t() + _bias(p, [f + "up"])
    y = torch.nn.functional.silu(g) * u
    dg, du = (sum_slack(av, v, v.shape[1]) + 2.0 ** -22 * t.abs() for v, t in ((wg, g), (wu, u)))
    slack = 1.1 * dg * u.abs() + torch.nn.functional.silu(g).abs() * du + 2.0 ** -18 * y.abs()
    assert_held_near(codes, scales, _f64(y), _f64(slack))


def checks(sess, block):
    """(what, check(params)) of one block's FP8 launches."""
    prefix, stream, tokens, first, last, b = block
    dim, hidden, a, f = sess.dim, sess.hidden, prefix + "attention.", prefix + "feed_forward."
    rows = lambda i, name: b[i][name][:tokens]
    op = lambda i, name, cols: _operand(b[i], name, tokens, cols)
    qkv = [a + n for n in ("query", "key", "value")]
    att = op(6, "rows8", dim)
    yield "attention norm", lambda p: check_norm(p, prefix + "attention_norm", sess.eps, rows(0, stream),
                                                 None if first else rows(0, "delta"), rows(1, stream),
                                                 *op(1, "rows8", dim)[:2])
    yield "qkv", lambda p: check_product(p, qkv, op(1, "rows8", dim), rows(2, "qkv"))
    codes, scales = o8.quantize(_f64(rows(5, "att")))
    np.testing.assert_array_equal(att[0].cpu().numpy(), codes)
    np.testing.assert_array_equal(att[1].cpu().numpy(), o8.lay_out(scales))
    yield "output", lambda p: check_product(p, [a + "output"], att, rows(7, "delta"))
    yield "feed-forward norm", lambda p: check_norm(p, prefix + "feed_forward_norm", sess.eps, rows(7, stream),
                                                    rows(7, "delta"), rows(8, stream), *op(8, "rows8", dim)[:2])
    yield "gated", lambda p: check_gated(p, f, op(8, "rows8", dim), *op(9, "act8", hidden)[:2])
    act = op(9, "act8", hidden)
    yield "down", lambda p: check_product(p, [f + "down"], act, rows(10, stream if last else "delta"),
                                          rows(9, stream) if last else None)


@pytest.mark.parametrize("tag", sorted(recipes.DECODER_CASES))
def test_every_launch_of_a_step(tag, monkeypatch):
    params = recipes.decoder_params(tag)
    sess, log = _recorded(tag, monkeypatch)
    for block in _blocks(sess, log):
        for what, check in checks(sess, block):
            try:
                check(params)
            except AssertionError as error:
                raise AssertionError(f"{block[0]} {what}") from error


def test_planted_faults_are_refused(monkeypatch):
    """With one parameter of the oracle lost, swapped or not held in 8 bits, the launch that uses it is refused."""
    params = recipes.decoder_params("s")
    sess, log = _recorded("s", monkeypatch)
    for block in _blocks(sess, log):
        prefix = block[0]
        a, f = prefix + "attention.", prefix + "feed_forward."
        uses = {"attention norm": [prefix + "attention_norm"], "feed-forward norm": [prefix + "feed_forward_norm"],
                "qkv": [a + "query", a + "key", a + "value"], "output": [a + "output"], "gated": [f + "gate", f + "up"],
                "down": [f + "down"]}
        for what, check in checks(sess, block):
            for name in uses[what]:
                faults = [{name + ".weight": np.roll(params[name + ".weight"], 1, 0)}]
                if "norm" not in what:
                    faults.append({name + ".bias": np.zeros_like(params[name + ".bias"])})
                for fault in faults:
                    with pytest.raises(AssertionError):
                        check({**params, **fault})
            if "norm" not in what:
                with monkeypatch.context() as patch:
                    patch.setattr(o8, "quantize_weight", lambda w: (w, None))
                    patch.setattr(o8, "values", lambda w, _: w)
                    with pytest.raises(AssertionError):
                        check(params)


def test_buffers_are_those_of_the_linears():
    """Neither form of the session holds the other one's activation buffers."""
    fp8, bf16 = _session("s", linears="fp8_block"), _session("s")
    assert not hasattr(fp8, "xn") and not hasattr(bf16, "rows8") and not hasattr(bf16, "delta")
