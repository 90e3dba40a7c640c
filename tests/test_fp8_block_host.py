"""Block-scaled FP8 on the host: the definition's own properties, the layouts
and the refusals of the C entry points (CPU, nothing is launched)."""
import numpy as np
import pytest
import torch

from oracle import fp8_block as oracle


def test_scale_byte_is_the_smallest_that_holds_amax():
    amax = np.concatenate([[0.0, 1e-45, 2.0 ** -126, 448.0, np.nextafter(448.0, 1e9), 3.38e38],
                           np.exp2(np.linspace(-120, 127, 1000)), 1.75 * np.exp2(np.arange(-110.0, 120.0))])
    e = oracle.scale_byte(amax).astype(np.float64)
    assert (amax <= 448 * np.exp2(e - 127)).all()
    assert ((e == 1) | (amax > 448 * np.exp2(e - 128))).all()
    assert (oracle.scale_byte([np.inf, np.nan]) == 255).all()


def test_scale_byte_by_bits():
    """The kernels' integer form: the add carries into the exponent exactly when the mantissa is above 1.75."""
    rs = np.random.RandomState(0)
    bits = np.concatenate([rs.randint(0, 0x7f800000, 200000),
                           (np.arange(1, 255)[:, None] * 0x800000 + np.array([0, 0x5fffff, 0x600000, 0x600001, 0x7fffff])).ravel()])
    amax = bits.astype(np.uint32).view(np.float32).astype(np.float64)
    e = np.maximum((bits + 0x1fffff >> 23) - 8, 1)
    np.testing.assert_array_equal(e, oracle.scale_byte(amax))


def test_encode_matches_torch():
    v = np.concatenate([np.linspace(-448, 448, 20001), oracle._GRID, (oracle._GRID[1:] + oracle._GRID[:-1]) / 2])
    v = v.astype(np.float32)
    got = torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(oracle.encode(v), got)
    np.testing.assert_array_equal(oracle.decode(got), torch.from_numpy(got).view(torch.float8_e4m3fn).float().numpy())


@pytest.mark.parametrize("rows,cols", [(1, 16), (130, 528), (128, 512), (257, 1040)])
def test_scale_layout(rows, cols):
    from recavsr_b200.runtime import fp8_block
    rs = np.random.RandomState(rows)
    e = rs.randint(40, 200, (rows, -(-cols // 128))).astype(np.uint8)
    flat = torch.from_numpy(oracle.lay_out(e))
    assert flat.numel() == fp8_block.scale_numel(rows, cols)
    np.testing.assert_array_equal(fp8_block.scale_bytes(flat, rows, cols).numpy(), e)
    codes = torch.from_numpy(rs.randint(0, 127, (rows, cols)).astype(np.uint8))
    np.testing.assert_array_equal(fp8_block.dequantize(codes, flat).numpy(),
                                  oracle.values(codes.numpy(), e).astype(np.float32))


def test_scales_size_entry_point():
    from recavsr_b200 import _lib
    from recavsr_b200.runtime import fp8_block
    for rows, cols in ((1, 16), (128, 512), (129, 528), (7040, 14336)):
        assert _lib.library().rc_fp8_block_scales(rows, cols) == fp8_block.scale_numel(rows, cols)


def test_interleave_gate_up():
    from recavsr_b200.runtime import fp8_block
    gate = torch.arange(144 * 2.0).reshape(144, 2)
    both = fp8_block.interleave_gate_up(gate, -gate)
    assert both.shape == (512, 2)
    assert torch.equal(both[:128], gate[:128]) and torch.equal(both[128:256], -gate[:128])
    assert torch.equal(both[256:272], gate[128:]) and torch.equal(both[384:400], -gate[128:])
    assert not both[272:384].any() and not both[400:].any()
    assert fp8_block.interleave_gate_up(gate[:, 0], gate[:, 1]).shape == (512,)


def test_cpu_tensors_are_refused():
    from recavsr_b200.runtime import fp8_block
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    codes, scales = torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    for call in (lambda: fp8_block.quantize(x), lambda: fp8_block.quantize_weight(x),
                 lambda: fp8_block.rms_norm_quantize(x, torch.ones(64), 1e-5),
                 lambda: fp8_block.mm(codes, codes, scales, scales),
                 lambda: fp8_block.swiglu_mm(codes, codes, scales, scales)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    from recavsr_b200 import _fp8_block
    with pytest.raises(RuntimeError, match="expected 8 arguments"):
        _fp8_block.mm(codes, codes, scales, scales)
    with pytest.raises(ValueError, match="tensor"):
        fp8_block.quantize("x")


def test_entry_points_reject_bad_arguments():
    from recavsr_b200 import _lib
    p = 4096          # an aligned address that no call below gets to read
    for name in ("rc_fp8_block_quantize", "rc_fp8_block_quantize_weight"):
        for args in ((p, 3, 4, 64, 64, p, p), (p, 1, 4, 40, 40, p, p), (p, 1, -1, 64, 64, p, p),
                     (p, 1, 4, 64, 48, p, p), (p, 1, 4, 64, 68, p, p), (None, 1, 4, 64, 64, p, p),
                     (p, 1, 4, 64, 64, p + 8, p), (p, 1, 4, 64, 64, p, None)):
            with pytest.raises(ValueError, match=name):
                _lib.call(name, *args, None)
        _lib.call(name, None, 1, 0, 64, 64, None, None, None)       # no rows: nothing to do
    norm = "rc_fp8_block_rms_norm"
    for args in ((p, 64, None, 0, 1, 4, 64, None, 1e-5, None, p, p), (p, 64, p, 64, 1, 4, 64, p, 1e-5, None, p, p),
                 (p, 64, p, 60, 1, 4, 64, p, 1e-5, p, p, p), (p, 64, None, 0, 1, 4, 72, p, 1e-5, None, p, p),
                 (p, 16400, None, 0, 1, 4, 16400, p, 1e-5, None, p, p)):
        with pytest.raises(ValueError, match=norm):
            _lib.call(norm, *args, None)
    gemm = "rc_fp8_block_gemm"
    good = dict(a=p, lda=64, sa=p, b=p, ldb=64, sb=p, bias=None, m=4, n=8, k=64, t=1, r=None, ldr=0, o=p, ldo=8)
    for change in (dict(k=40), dict(n=0), dict(m=-1), dict(lda=48), dict(ldb=72), dict(t=0), dict(a=None),
                   dict(sb=p + 4), dict(bias=p + 4), dict(o=None), dict(ldo=7), dict(r=p, ldr=7), dict(o=p + 1)):
        with pytest.raises(ValueError, match=gemm):
            _lib.call(gemm, *{**good, **change}.values(), None)
    _lib.call(gemm, *{**good, "m": 0}.values(), None)
    gated = "rc_fp8_block_swiglu_gemm"
    good = dict(a=p, lda=64, sa=p, b=p, ldb=64, sb=p, bias=None, m=4, h=16, k=64, c=p, s=p)
    for change in (dict(h=24), dict(h=0), dict(k=8), dict(c=None), dict(s=p + 8), dict(lda=32)):
        with pytest.raises(ValueError, match=gated):
            _lib.call(gated, *{**good, **change}.values(), None)
    _lib.call(gated, *{**good, "m": 0}.values(), None)
