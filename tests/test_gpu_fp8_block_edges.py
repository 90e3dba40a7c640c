"""Block-scaled FP8 operators at their edges: few rows with K over a cluster,
gates far below zero, special values, strides and middle row counts of the gated
product.

Tolerances of the products: tests/test_gpu_fp8_block.py."""
import pytest
import torch

from tests.test_gpu_fp8_block import (activations, assert_held_near, assert_rounded_from, check_mm, check_swiglu, f64,
                                      held, operands, sum_slack)
from tests.util import assert_no_device_error

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- few rows, K over a cluster
@pytest.mark.parametrize("m", [1, 7, 16, 17, 32])
@pytest.mark.parametrize("n,k", [(128, 128), (512, 256), (512, 512), (1000, 1024), (3072, 1024), (128, 4096)])
def test_mm_few_rows_short_ranges(m, n, k):
    """One to a few k-tiles for each CTA of a cluster of 1 to 8: a CTA sends its
    partials to the others as early as it can."""
    check_mm(m, n, k)
    assert_no_device_error()


@pytest.mark.parametrize("m", [1, 16, 17, 32])
@pytest.mark.parametrize("h,k", [(128, 256), (2048, 512), (1040, 1024)])
def test_swiglu_few_rows_short_ranges(m, h, k):
    check_swiglu(m, h, k)
    assert_no_device_error()


@pytest.mark.parametrize("n,k", [(512, 512), (3072, 1024), (14336, 256)])
def test_few_rows_back_to_back(n, k):
    """Launches queued back to back: clusters start while earlier ones end, and every result is the same."""
    from recavsr_b200.runtime import fp8_block
    (ac, asc), (bc, bsc), av, bv = operands(3, n, k, 31)
    outs = [fp8_block.mm(ac, bc, asc, bsc) for _ in range(200)]
    assert_rounded_from(outs[0], av @ bv.t(), sum_slack(av, bv, k))
    for out in outs[1:]:
        assert torch.equal(out, outs[0])
    assert_no_device_error()


def _microseconds(call, launches=20, times=7):
    """Least device time of one launch out of a graph of them."""
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(launches):
            call()
    best = float("inf")
    for _ in range(times):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        graph.replay()
        end.record()
        end.synchronize()
        best = min(best, begin.elapsed_time(end) * 1e3 / launches)
    return best


@pytest.mark.parametrize("fits,more,k", [(4096, 8192, 512), (1792, 2048, 4096)])
def test_few_rows_run_in_one_wave(fits, more, k):
    """Gated tiles of 32 rows have an SM to themselves: more tiles than clusters
    find room for must mean smaller clusters, not a second wave (twice the time)."""
    from recavsr_b200.runtime import fp8_block
    took = []
    for h in (fits, more):
        ac, asc = fp8_block.quantize(activations(32, k, torch.bfloat16, 51))
        wc, wsc = fp8_block.quantize_weight(torch.randn(2 * h, k, device="cuda") / k ** 0.5)
        took.append(_microseconds(lambda: fp8_block.swiglu_mm(ac, wc, asc, wsc)))
    assert took[1] < 1.5 * took[0], took


# ---------------------------------------------------------------- gates far from zero
# Instruction errors of silu(g) u = g / (1 + t) * p * u * p with t = s^2 = exp(-|g|) and p = s below zero, else 1:
# s carries 2^-22 of the exponential and |g| / 2 (2^-24 + 2^-26) of its rounded argument, both twice in p p and once
# more at most through 1 + t; the reciprocal and five roundings add 2^-23 + 5 2^-24: under 2^-19 + |g| 2^-23.
def gated_reference(g, u, dg, du):
    """silu(g) u in 64 bits, and how far off it may be when g and u are known to within dg and du."""
    sigma = torch.sigmoid(g)
    y = g * sigma * u
    # |silu'| <= sigma (1 + |g|) and sigma grows by at most exp(dg) over dg
    slack = 1.01 * sigma * (1 + g.abs()) * dg * u.abs() + (g * sigma).abs() * du
    return y, slack + (2.0 ** -19 + g.abs() * 2.0 ** -23) * y.abs() + 2.0 ** -148


@pytest.mark.parametrize("m", [2, 20, 40, 300])
def test_swiglu_gates_far_below_zero(m):
    """Whole blocks of 128 outputs with gates about -10 to -150 (and one of large
    positive ones): fp32 holds exp(-|g|) of the first five, and the square root
    of the others'; an 8-bit block holds values down to 2^-136."""
    from recavsr_b200.runtime import fp8_block
    k, gates = 256, [-10.0, -30.0, -60.0, -80.0, -86.0, -90.0, -93.0, -150.0, 40.0]
    h = 128 * len(gates)
    gen = torch.Generator("cuda").manual_seed(41)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    ac, asc = fp8_block.quantize(rand(m, k))
    wc, wsc = fp8_block.quantize_weight(fp8_block.interleave_gate_up(rand(h, k) / k ** 0.5, rand(h, k) / k ** 0.5))
    bg = torch.tensor(gates, device="cuda").repeat_interleave(128)
    bu = rand(h)
    got = fp8_block.swiglu_mm(ac, wc, asc, wsc, fp8_block.interleave_gate_up(bg, bu), features=h)
    av = fp8_block.dequantize(ac, asc).double()
    wv = fp8_block.dequantize(wc, wsc).double().view(-1, 2, 128, k)
    gv, uv = wv[:, 0].reshape(-1, k), wv[:, 1].reshape(-1, k)
    g, u = av @ gv.t() + bg.double(), av @ uv.t() + bu.double()
    y, slack = gated_reference(g, u, *(sum_slack(av, v, k) + 2.0 ** -22 * t.abs() for v, t in ((gv, g), (uv, u))))
    assert_held_near(*got, f64(y), f64(slack))
    assert_no_device_error()


# ---------------------------------------------------------------- gated product
@pytest.mark.parametrize("m", [3, 30, 200])
def test_swiglu_special_values(m):
    """A NaN or an infinity of the operands marks the row's blocks that it reaches; zero rows stay zero."""
    from recavsr_b200.runtime import fp8_block
    k, h = 256, 256
    x = activations(m, k, torch.float32, 42)
    clean = x.clone()
    clean[0] = 0
    x[0], x[1, 3], x[2, 200] = 0, float("nan"), float("inf")
    w = fp8_block.quantize_weight(fp8_block.interleave_gate_up(*activations(2 * h, k, torch.float32, 43).chunk(2)))
    (ac, asc), (bc, bsc) = fp8_block.quantize(x), fp8_block.quantize(clean)
    codes, scales = fp8_block.swiglu_mm(ac, w[0], asc, w[1])
    want, want_scales = fp8_block.swiglu_mm(bc, w[0], bsc, w[1])
    c, e = held(codes, scales)
    wc, we = held(want, want_scales)
    assert not (c[0] & 0x7f).any() and (e[0] == 1).all()
    for row in (1, 2):
        assert (c[row] == 0x7f).all() and (e[row] == 255).all()
    rest = [i for i in range(m) if i not in (1, 2)]
    assert (c[rest] == wc[rest]).all() and (e[rest] == we[rest]).all()


@pytest.mark.parametrize("m,h,k", [(33, 1024, 4096), (100, 1040, 2064), (256, 2048, 4096), (520, 528, 1536),
                                   (900, 1024, 2048)])
def test_swiglu_middle_rows(m, h, k):
    check_swiglu(m, h, k)
    assert_no_device_error()


@pytest.mark.parametrize("m", [5, 200])
def test_swiglu_strided_codes(m):
    """Codes as columns of wider buffers, on and off 16 bytes."""
    from recavsr_b200.runtime import fp8_block
    ac, asc = fp8_block.quantize(activations(m, 256, torch.float32, 44))
    wc, wsc = fp8_block.quantize_weight(activations(256, 256, torch.float32, 45))
    want = fp8_block.swiglu_mm(ac, wc, asc, wsc)
    for cols, at in ((512, 64), (300, 3)):
        wide, weight = (torch.zeros(t.shape[0], cols, dtype=torch.uint8, device="cuda") for t in (ac, wc))
        wide[:, at:at + 256], weight[:, at:at + 256] = ac, wc
        got = fp8_block.swiglu_mm(wide[:, at:at + 256], weight[:, at:at + 256], asc, wsc)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------- gradients and torch.compile
def test_lost_gradients_raise():
    """No operator has a backward pass: a result whose gradient would be asked for
    says so in backward instead of standing there as a constant."""
    from recavsr_b200.runtime import fp8_block
    x, w = activations(5, 128, torch.bfloat16, 61), torch.ones(128, device="cuda")
    (ac, asc), (bc, bsc) = fp8_block.quantize(x), fp8_block.quantize_weight(activations(64, 128, torch.bfloat16, 62))
    bias, res = torch.zeros(64, device="cuda"), torch.zeros(5, 64, dtype=torch.bfloat16, device="cuda")
    leaf = lambda t: t.clone().requires_grad_()
    lin = fp8_block.BlockFP8Linear(torch.nn.Linear(128, 64, device="cuda", dtype=torch.bfloat16))
    calls = [(lambda: fp8_block.mm(ac, bc, asc, bsc, leaf(bias)), lambda: fp8_block.mm(ac, bc, asc, bsc, bias)),
             (lambda: fp8_block.mm(ac, bc, asc, bsc, residual=leaf(res)),
              lambda: fp8_block.mm(ac, bc, asc, bsc, residual=res)),
             (lambda: fp8_block.rms_norm_quantize(leaf(x), w, 1e-5, residual=x)[2],
              lambda: fp8_block.rms_norm_quantize(x, w, 1e-5, residual=x)[2]),
             (lambda: lin(leaf(x)), lambda: lin(x))]
    for call, plain in calls:
        got, want = call(), plain()
        assert torch.equal(got, want) and got.requires_grad and not want.requires_grad
        with pytest.raises(RuntimeError, match="no autograd formula"):
            got.float().sum().backward()
        with torch.no_grad():
            assert not call().requires_grad
    with pytest.raises(ValueError, match="gradient"):
        fp8_block.mm(ac, bc, asc, bsc, leaf(bias), out=res)
    with torch.no_grad():
        assert fp8_block.mm(ac, bc, asc, bsc, leaf(bias), out=res) is not None
    # codes are whole numbers: no gradient, and none promised
    gu = fp8_block.quantize_weight(activations(256, 128, torch.bfloat16, 67))
    for q in (fp8_block.quantize(leaf(x)), fp8_block.rms_norm_quantize(leaf(x), w, 1e-5)[:2],
              fp8_block.swiglu_mm(ac, gu[0], asc, gu[1], leaf(torch.zeros(256, device="cuda")))):
        assert not any(t.requires_grad for t in q)


@pytest.mark.parametrize("dynamic", [False, True])
def test_operators_compile(dynamic):
    """torch.compile(fullgraph=True) traces through all four, in-place products among them."""
    from recavsr_b200.runtime import fp8_block
    w = torch.ones(512, device="cuda")
    wo = fp8_block.quantize_weight(activations(512, 512, torch.bfloat16, 63))
    gu = fp8_block.quantize_weight(fp8_block.interleave_gate_up(*activations(416, 512, torch.bfloat16, 64).chunk(2)))
    down = fp8_block.quantize_weight(activations(512, 208, torch.bfloat16, 65))
    bias = torch.randn(512, device="cuda", generator=torch.Generator("cuda").manual_seed(66))

    def block(x, hidden):
        codes, scales, _ = fp8_block.rms_norm_quantize(x, w, 1e-5)
        delta = fp8_block.mm(codes, wo[0], scales, wo[1], bias)
        codes, scales, hidden = fp8_block.rms_norm_quantize(delta, w, 1e-5, residual=hidden)
        codes, scales = fp8_block.swiglu_mm(codes, gu[0], scales, gu[1], features=208)
        out = hidden.clone()
        fp8_block.mm(codes, down[0], scales, down[1], bias, residual=out, out=out)
        return out, codes, scales

    compiled = torch.compile(block, fullgraph=True, backend="aot_eager", dynamic=dynamic)
    with torch.inference_mode():
        for rows in (37, 300):
            x, r = activations(rows, 512, torch.bfloat16, rows), activations(rows, 512, torch.bfloat16, rows + 1)
            for got, want in zip(compiled(x, r), block(x, r)):
                assert torch.equal(got, want)


# ---------------------------------------------------------------- refusals
def test_other_eight_bit_types_are_refused():
    """Bytes of another 8-bit format read as E4M3 codes or E8M0 scales would give wrong products."""
    from recavsr_b200.runtime import fp8_block
    a, s = fp8_block.quantize(activations(4, 256, torch.bfloat16, 71))
    for t, ts in ((a.view(torch.float8_e4m3fn), s), (a, s.view(torch.float8_e8m0fnu))):
        assert torch.equal(fp8_block.mm(t, a, ts, s), fp8_block.mm(a, a, s, s))
    for dtype in (torch.float8_e5m2, torch.float8_e4m3fnuz, torch.int8, torch.bool):
        for call in (lambda: fp8_block.mm(a.view(dtype), a, s, s), lambda: fp8_block.mm(a, a.view(dtype), s, s),
                     lambda: fp8_block.swiglu_mm(a.view(dtype), a, s, s)):
            with pytest.raises(ValueError, match="float8_e4m3fn codes"):
                call()
    for dtype in (torch.float8_e4m3fn, torch.int8):
        for call in (lambda: fp8_block.mm(a, a, s.view(dtype), s), lambda: fp8_block.mm(a, a, s, s.view(dtype))):
            with pytest.raises(ValueError, match="float8_e8m0fnu scales"):
                call()


@pytest.mark.parametrize("m", [1, 6, 200])
def test_outputs_that_share_memory(m):
    """out may be the residual, or lie beside any input in one buffer, but not over it."""
    from recavsr_b200.runtime import fp8_block
    n = k = 128
    (ac, asc), (bc, bsc), _, _ = operands(m, n, k, 72)
    buffer = activations(m + 2, 3 * n, torch.bfloat16, 73)
    mm = lambda r, o, bias=None: fp8_block.mm(ac, bc, asc, bsc, bias, residual=r, out=o)
    fresh = lambda: buffer.clone()
    want = fp8_block.mm(ac, bc, asc, bsc, residual=buffer[:m, :n])
    for at in (n, 2 * n):                        # columns beside the residual's
        b = fresh()
        assert torch.equal(mm(b[:m, :n], b[:m, at:at + n]), want)
        assert torch.equal(b[:m, :n], buffer[:m, :n])
    b = fresh()
    assert torch.equal(mm(b[:m, :n], b[:m, :n]), want)
    b = fresh()
    for r, o in ((b[:m, :n], b[:m, 8:8 + n]), (b[:m, 8:8 + n], b[:m, :n]), (b[1:m + 1, :n], b[1:m + 1, n - 8:2 * n - 8])):
        with pytest.raises(ValueError, match="shares memory"):
            mm(r, o)
    flat = fresh().flatten()
    with pytest.raises(ValueError, match="shares memory"):
        mm(flat[:m * n].view(m, n), flat[n // 2:n // 2 + m * n].view(m, n))
    if m > 1:                                    # rows below the residual's, and one buffer in two strides
        for r, o in ((b[:m, :n], b[1:m + 1, :n]), (flat[:m * n].view(m, n), flat[:m * 2 * n].view(m, 2 * n)[:, :n])):
            with pytest.raises(ValueError, match="shares memory"):
                mm(r, o)
    raw = torch.zeros(4 * m * n + 4 * n, dtype=torch.uint8, device="cuda")
    raw[:m * k] = ac.flatten()
    codes, over = raw[:m * k].view(m, k), raw[:2 * m * n].view(torch.bfloat16).view(m, n)
    with pytest.raises(ValueError, match="shares memory"):
        fp8_block.mm(codes, bc, asc, bsc, out=over)
    with pytest.raises(ValueError, match="shares memory"):
        mm(None, over, raw[:4 * n].view(torch.float32))


@pytest.mark.parametrize("m", [3, 200])
def test_smallest_and_largest_scale_bytes(m):
    """Operands of others may hold scale byte 0 (2^-127); 254 is the largest (its
    values pass fp32, the products here do not)."""
    from recavsr_b200.runtime import fp8_block
    (ac, asc), (bc, bsc), _, _ = operands(m, 128, 256, 81)
    for a_byte, b_byte in ((0, 224), (254, 20), (1, 254)):
        sa, sb = (torch.where(s > 0, byte, 0).to(torch.uint8) for s, byte in ((asc, a_byte), (bsc, b_byte)))
        av, bv = (c.view(torch.float8_e4m3fn).double() * 2.0 ** (byte - 127) for c, byte in ((ac, a_byte), (bc, b_byte)))
        assert_rounded_from(fp8_block.mm(ac, bc, sa, sb), av @ bv.t(), sum_slack(av, bv, 256))
