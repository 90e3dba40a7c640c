"""The values that block-scaled FP8 codes and scale bytes stand for (CPU)."""
import numpy as np
import torch

from oracle import fp8_block as oracle


def test_every_scale_byte():
    """Byte e is 2^(e-127), the subnormal 2^-127 for 0 (which no quantizer here writes, but others do) and NaN for 255."""
    from recavsr_b200.runtime import fp8_block
    e = np.arange(256, dtype=np.uint8)[:, None]
    codes = np.full((256, 16), 0x38, np.uint8)                 # 1.0
    got = fp8_block.dequantize(torch.from_numpy(codes), torch.from_numpy(oracle.lay_out(e))).numpy()
    want = np.append(np.ldexp(1.0, np.arange(255) - 127), np.nan).astype(np.float32)
    np.testing.assert_array_equal(got, np.repeat(want[:, None], 16, 1))
