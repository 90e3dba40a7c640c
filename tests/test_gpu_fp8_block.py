"""Block-scaled FP8 operators on the GPU against the 64-bit definition
(oracle/fp8_block.py).

Tolerances. quantize is exact: its scaling is by powers of two. Elsewhere a
value y reaches the quantizer in fp32 with a relative error of at most DELTA
(a few roundings, a sum of squares of at most 16384 terms added in a tree of
fp32 partial sums of at most 32: under 64 * 2^-24), so a scale byte is that of
amax (1 +- DELTA) and a code is off by half an E4M3 step (2^-4 of the value, or
half of 2^-9 of the scale) plus DELTA. A product's terms are exact; summing K
of them in fp32 in K / 32 steps, each truncated once in the dot product and
once in the accumulator, is off by at most 2 (K / 32 + 1) 2^-23 sum|a w|; bias
and residual add 2^-23 of each. The output is that sum rounded once, so it lies
between the roundings of the lowest and the highest sum it may be."""
import numpy as np
import pytest
import torch

from oracle import fp8_block as oracle
from tests.util import assert_no_device_error

pytestmark = pytest.mark.gpu

DELTA = 64 * 2.0 ** -24
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def activations(m, n, dtype, seed):
    rs = np.random.RandomState(seed)
    x = rs.standard_normal((m, n)) * np.exp(0.5 * rs.standard_normal(n)) * np.exp(0.3 * rs.standard_normal((m, 1)))
    x[:, rs.rand(n) < 0.02] *= 12
    return torch.from_numpy(x.astype(np.float32)).to("cuda", dtype)


def f64(t):
    return t.detach().double().cpu().numpy()


def held(codes, scales):
    """(codes, scale bytes [rows, blocks]) on the host, padding checked."""
    from recavsr_b200.runtime import fp8_block
    m, n = codes.shape
    e = fp8_block.scale_bytes(scales, m, n).cpu().numpy()
    np.testing.assert_array_equal(scales.cpu().numpy(), oracle.lay_out(e))
    return codes.cpu().numpy(), e


def assert_held_near(codes, scales, y, slack):
    """codes / scales hold y, itself known to within slack (absolute, per value)."""
    c, e = held(codes, scales)
    blocks = lambda v: oracle._blocks(v).max(-1)
    amax, room = blocks(np.abs(y)), blocks(np.broadcast_to(slack, y.shape))
    low, high = oracle.scale_byte(np.maximum(amax - room, 0)), oracle.scale_byte(amax + room)
    assert ((low <= e) & (e <= high)).all()
    v = oracle.values(c, e)
    s = np.repeat(np.exp2(e.astype(np.float64) - 127), 128, 1)[:, :y.shape[1]]
    err = np.abs(v - y)
    assert (err <= np.maximum(np.abs(y) * (1 + 2.0 ** -4) * 2.0 ** -4, s * 2.0 ** -10) + slack * 1.125).all(), err.max()


# ---------------------------------------------------------------- quantizers
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 16), (3, 112), (17, 128), (33, 144), (130, 528), (200, 2048), (5, 14336)])
def test_quantize(m, k, dtype):
    from recavsr_b200.runtime import fp8_block
    x = activations(m, k, DTYPES[dtype], 1)
    c, e = held(*fp8_block.quantize(x))
    rc, re = oracle.quantize(f64(x))
    np.testing.assert_array_equal(e, re)
    np.testing.assert_array_equal(c, rc)


def test_quantize_extremes():
    """Zero blocks, blocks at a scale's edge, subnormals, the type's largest, infinities and NaN."""
    from recavsr_b200.runtime import fp8_block
    rs = np.random.RandomState(3)
    x = rs.standard_normal((64, 256)).astype(np.float32)
    x[0] = 0
    x[1] = -0.0
    x[2] *= np.float32(1e-42)
    x[3] *= np.float32(1e37)
    x[4, 5], x[4, 6] = 3.4e38, -3.4e38
    x[5, :128] = 448.0
    x[6, 0] = np.nextafter(np.float32(448), np.float32(1e9))
    x[7, 0], x[7, 128] = 1.75 * 2.0 ** 20, np.nextafter(np.float32(1.75 * 2.0 ** 20), np.float32(1e9))
    x[8, 3], x[9, 200], x[10, 0] = np.inf, -np.inf, np.nan
    x[11] = 2.0 ** -127
    for j in range(20, 40):
        x[j] = np.exp2(rs.uniform(-140, 120)) * x[j]
    t = torch.from_numpy(x).cuda()
    c, e = held(*fp8_block.quantize(t))
    rc, re = oracle.quantize(x)
    np.testing.assert_array_equal(e, re)
    np.testing.assert_array_equal(c, rc)
    assert (e[8, 0], e[8, 1] != 255, e[9, 1], e[10, 0]) == (255, True, 255, 255) and (c[8, :128] == 0x7f).all()


def test_quantize_every_bf16_value():
    from recavsr_b200.runtime import fp8_block
    bits = np.arange(65536, dtype=np.uint32).astype(np.uint16)
    x = torch.from_numpy(bits.view(np.int16)).view(torch.bfloat16).reshape(512, 128).cuda()
    c, e = held(*fp8_block.quantize(x))
    rc, re = oracle.quantize(f64(x))
    np.testing.assert_array_equal(e, re)
    np.testing.assert_array_equal(c, rc)


@pytest.mark.parametrize("n,k", [(1, 16), (128, 128), (129, 144), (300, 528), (48, 768)])
def test_quantize_weight(n, k):
    from recavsr_b200.runtime import fp8_block
    w = activations(n, k, torch.bfloat16, 2)
    c, e = held(*fp8_block.quantize_weight(w))
    rc, re = oracle.quantize_weight(f64(w))
    np.testing.assert_array_equal(e, re)
    np.testing.assert_array_equal(c, rc)


@pytest.mark.parametrize("layout", ["columns", "odd stride", "transposed", "offset"])
def test_quantize_layouts(layout):
    from recavsr_b200.runtime import fp8_block
    base = activations(96, 400, torch.bfloat16, 4)
    x = {"columns": base[:, 128:336], "odd stride": base.flatten()[:60 * 401].view(60, 401)[:, :208],
         "transposed": base[:, :208].t()[:, :80], "offset": base[:, 3:3 + 208]}[layout]
    c, e = held(*fp8_block.quantize(x))
    rc, re = oracle.quantize(f64(x))
    np.testing.assert_array_equal(c, rc)
    np.testing.assert_array_equal(e, re)


# ---------------------------------------------------------------- norm
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n", [(1, 16), (3, 144), (130, 512), (9, 528), (17, 1024), (5, 1040), (33, 2048), (4, 3072),
                                 (3, 4112), (2, 8192), (3, 12304), (2, 16384)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_rms_norm(m, n, dtype, with_residual):
    from recavsr_b200.runtime import fp8_block
    dt = DTYPES[dtype]
    x = activations(m, n, dt, 5)
    r = activations(m, n, dt, 6) if with_residual else None
    w = 1 + 0.1 * torch.randn(n, device="cuda", generator=torch.Generator("cuda").manual_seed(7))
    codes, scales, hidden = fp8_block.rms_norm_quantize(x, w, 1e-5, residual=r)
    y, _ = oracle.rms_norm(f64(x), f64(w), 1e-5, None if r is None else f64(r))
    assert_held_near(codes, scales, y, np.abs(y) * DELTA)
    if r is None:
        assert hidden is None
    else:
        assert torch.equal(hidden, (x.float() + r.float()).to(dt))
    assert_no_device_error()


def test_rms_norm_strides_and_weight_types():
    from recavsr_b200.runtime import fp8_block
    x, r = activations(40, 800, torch.bfloat16, 8)[:, 16:16 + 512], activations(40, 1024, torch.bfloat16, 9)[:, 8:520]
    w = (1 + 0.1 * torch.randn(513, device="cuda")).bfloat16()[1:]
    codes, scales, hidden = fp8_block.rms_norm_quantize(x, w, 1e-5, residual=r)
    y, _ = oracle.rms_norm(f64(x), f64(w), 1e-5, f64(r))
    assert_held_near(codes, scales, y, np.abs(y) * DELTA)
    assert torch.equal(hidden, (x.float() + r.float()).bfloat16())


def test_rms_norm_special_rows():
    """Zero rows stay zero; a NaN or an infinity marks its row, and no other."""
    from recavsr_b200.runtime import fp8_block
    x = activations(8, 256, torch.float32, 10)
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 200] = float("inf")
    w = torch.ones(256, device="cuda")
    codes, scales, _ = fp8_block.rms_norm_quantize(x, w, 1e-5)
    c, e = held(codes, scales)
    assert not c[1].any() and (e[1] == 1).all()
    assert (e[2] == 255).all() and (c[2] == 0x7f).all()
    assert e[3, 1] == 255                       # inf * 0 is a NaN in its own block; the rest of the row is 0
    rest = [0, 1, 4, 5, 6, 7]
    y, _ = oracle.rms_norm(f64(x[rest]), f64(w), 1e-5)
    back = fp8_block.quantize(x[rest])
    assert back[0].shape == (6, 256)
    got, se, _ = fp8_block.rms_norm_quantize(x[rest].contiguous(), w, 1e-5)
    np.testing.assert_array_equal(c[rest], got.cpu().numpy())
    assert_held_near(got, se, y, np.abs(y) * DELTA)


# ---------------------------------------------------------------- products
def operands(m, n, k, seed):
    """Codes and scales of both operands (the oracle's, uploaded), and their 64-bit values."""
    from recavsr_b200.runtime import fp8_block
    a = fp8_block.quantize(activations(m, k, torch.float32, seed))
    rs = np.random.RandomState(seed + 100)
    w = torch.from_numpy((rs.standard_normal((n, k)) / k ** 0.5).astype(np.float32)).cuda()
    b = fp8_block.quantize_weight(w)
    value = lambda q: fp8_block.dequantize(*q).double()
    return a, b, value(a), value(b)


def sum_slack(av, bv, k):
    return 2 * (k / 32 + 1) * 2.0 ** -23 * (av.abs() @ bv.abs().t())


def assert_rounded_from(out, ref, slack):
    low, high = (ref - slack).to(out.dtype), (ref + slack).to(out.dtype)
    bad = ~((low <= out) & (out <= high))
    assert not bad.any(), (int(bad.sum()), out[bad][:4], ref[bad][:4], slack[bad][:4])


def check_mm(m, n, k, dtype=torch.bfloat16, bias=True, residual=True, seed=11):
    from recavsr_b200.runtime import fp8_block
    (ac, asc), (bc, bsc), av, bv = operands(m, n, k, seed)
    g = torch.Generator("cuda").manual_seed(seed)
    bt = torch.randn(n, device="cuda", generator=g) if bias else None
    rt = torch.randn(m, n, device="cuda", generator=g).to(dtype) if residual else None
    out = fp8_block.mm(ac, bc, asc, bsc, bt, residual=rt, dtype=dtype)
    ref, slack = av @ bv.t(), sum_slack(av, bv, k)
    for extra in (bt, rt):
        if extra is not None:
            ref = ref + extra.double()
            slack = slack + 2.0 ** -23 * (extra.double().abs() + ref.abs())
    assert out.dtype == dtype and out.shape == (m, n)
    assert_rounded_from(out, ref, slack)


@pytest.mark.parametrize("k", [16, 48, 128, 144, 512, 528, 640, 2064])
@pytest.mark.parametrize("m,n", [(1, 128), (2, 47), (16, 48), (17, 256), (130, 129)])
def test_mm_lengths(m, n, k):
    check_mm(m, n, k)
    assert_no_device_error()


@pytest.mark.parametrize("m", [1, 3, 8, 15, 16, 31, 33, 64, 65, 100, 127, 128, 129, 200, 255, 257, 400, 1000])
@pytest.mark.parametrize("n", [1, 96, 300, 768])
def test_mm_rows(m, n):
    check_mm(m, n, 576)
    assert_no_device_error()


@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(1, 512, 512), (40, 200, 1024), (300, 513, 256)])
def test_mm_epilogues(m, n, k, dtype, bias, residual):
    check_mm(m, n, k, dtype, bias, residual)


@pytest.mark.parametrize("m,n,k", [(1, 3072, 14336), (24, 3072, 14336), (3520, 768, 512), (1759, 3072, 3072),
                                   (5000, 2048, 1024), (2500, 4096, 2048), (14080, 512, 2048), (640, 14336, 3072)])
def test_mm_large(m, n, k):
    check_mm(m, n, k)
    assert_no_device_error()


def test_mm_no_rows():
    from recavsr_b200.runtime import fp8_block
    a = fp8_block.quantize(torch.zeros(0, 256, dtype=torch.bfloat16, device="cuda"))
    b = fp8_block.quantize_weight(torch.ones(64, 256, dtype=torch.bfloat16, device="cuda"))
    assert a[0].shape == (0, 256) and a[1].numel() == 0
    assert fp8_block.mm(a[0], b[0], a[1], b[1]).shape == (0, 64)
    n = fp8_block.rms_norm_quantize(torch.zeros(0, 256, device="cuda"), torch.ones(256, device="cuda"), 1e-5)
    assert n[0].shape == (0, 256)


@pytest.mark.parametrize("m", [5, 200])
def test_mm_strided_operands_and_outputs(m):
    """Codes as columns of a wider buffer, out and residual with their own strides, out = residual."""
    from recavsr_b200.runtime import fp8_block
    (ac, asc), (bc, bsc), av, bv = operands(m, 96, 256, 12)
    wide = torch.zeros(m, 512, dtype=torch.uint8, device="cuda")
    wide[:, 64:320] = ac
    ref = fp8_block.mm(ac, bc, asc, bsc)
    assert torch.equal(fp8_block.mm(wide[:, 64:320], bc, asc, bsc), ref)
    odd = torch.zeros(m, 300, dtype=torch.uint8, device="cuda")
    odd[:, 3:259] = ac
    assert torch.equal(fp8_block.mm(odd[:, 3:259], bc, asc, bsc), ref)
    for pad, shift in ((32, 8), (5, 1)):
        buf = torch.full((m, 96 + pad), 7.0, dtype=torch.bfloat16, device="cuda")
        got = fp8_block.mm(ac, bc, asc, bsc, out=buf[:, shift:shift + 96])
        assert torch.equal(got, ref) and got.data_ptr() == buf[:, shift:].data_ptr()
        assert (buf[:, :shift] == 7).all() and (buf[:, shift + 96:] == 7).all()
    r = torch.randn(m, 96, device="cuda").bfloat16()
    want = fp8_block.mm(ac, bc, asc, bsc, residual=r)
    rr = torch.zeros(m, 104, dtype=torch.bfloat16, device="cuda")
    rr[:, 8:] = r
    assert torch.equal(fp8_block.mm(ac, bc, asc, bsc, residual=rr[:, 8:]), want)
    inplace = r.clone()
    fp8_block.mm(ac, bc, asc, bsc, residual=inplace, out=inplace)
    assert torch.equal(inplace, want)


@pytest.mark.parametrize("m", [4, 150])
def test_mm_nan_stays_in_its_row(m):
    from recavsr_b200.runtime import fp8_block
    x = activations(m, 384, torch.float32, 13)
    clean = x.clone()
    x[1, 130], x[2, 5] = float("nan"), float("inf")
    w = fp8_block.quantize_weight(activations(200, 384, torch.float32, 14))
    q, qc = fp8_block.quantize(x), fp8_block.quantize(clean)
    out, ref = fp8_block.mm(q[0], w[0], q[1], w[1]), fp8_block.mm(qc[0], w[0], qc[1], w[1])
    assert out[1].isnan().all() and out[2].isnan().all()
    keep = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(out[keep], ref[keep])


def test_mm_scale_range():
    """Scales from 2^-60 to 2^60 side by side in one row: each block is weighted by its own."""
    from recavsr_b200.runtime import fp8_block
    k = 128 * 9
    x = activations(20, k, torch.float32, 15)
    power = torch.tensor([-60, 60, -3, 0, 14, -28, 40, -41, 7], device="cuda", dtype=torch.float32)
    x = x * torch.exp2(power).repeat_interleave(128)
    a = fp8_block.quantize(x)
    for j in range(9):                          # a weight that reads one block only
        w = torch.zeros(64, k, device="cuda")
        w[:, 128 * j:128 * (j + 1)] = torch.randn(64, 128, device="cuda")
        b = fp8_block.quantize_weight(w)
        out = fp8_block.mm(a[0], b[0], a[1], b[1])
        av, bv = fp8_block.dequantize(*a).double(), fp8_block.dequantize(*b).double()
        av = av * (torch.arange(k, device="cuda") // 128 == j)
        assert_rounded_from(out, av @ bv.t(), sum_slack(av, bv, k))


# ---------------------------------------------------------------- gated product
def check_swiglu(m, h, k, bias=True, seed=16):
    from recavsr_b200.runtime import fp8_block
    rs = np.random.RandomState(seed)
    gate, up = (torch.from_numpy((rs.standard_normal((h, k)) / k ** 0.5).astype(np.float32)).cuda() for _ in range(2))
    bg, bu = (torch.from_numpy((0.5 * rs.standard_normal(h)).astype(np.float32)).cuda() for _ in range(2))
    x = activations(m, k, torch.float32, seed + 1)
    ac, asc = fp8_block.quantize(x)
    wc, wsc = fp8_block.quantize_weight(fp8_block.interleave_gate_up(gate, up))
    bt = fp8_block.interleave_gate_up(bg, bu) if bias else None
    codes, scales = fp8_block.swiglu_mm(ac, wc, asc, wsc, bt, features=h)
    av = fp8_block.dequantize(ac, asc).double()
    wv = fp8_block.dequantize(wc, wsc).double().view(-1, 2, 128, k)
    gv, uv = wv[:, 0].reshape(-1, k)[:h], wv[:, 1].reshape(-1, k)[:h]
    g, u = av @ gv.t(), av @ uv.t()
    if bias:
        g, u = g + bg.double(), u + bu.double()
    y = torch.nn.functional.silu(g) * u
    # d silu(g) <= 1.1 |dg|; the gate and up sums carry sum_slack, the rest a few fp32 roundings
    dg, du = (sum_slack(av, v, k) + 2.0 ** -22 * t.abs() for v, t in ((gv, g), (uv, u)))
    slack = 1.1 * dg * u.abs() + torch.nn.functional.silu(g).abs() * du + 2.0 ** -20 * y.abs() + 1e-30
    assert_held_near(codes, scales, f64(y), f64(slack))


@pytest.mark.parametrize("m", [1, 2, 9, 16, 17, 40, 64, 100, 128, 129, 200, 300])
@pytest.mark.parametrize("h,k", [(128, 128), (144, 80), (512, 576)])
def test_swiglu(m, h, k):
    check_swiglu(m, h, k)
    assert_no_device_error()


@pytest.mark.parametrize("m,h,k", [(16, 2048, 512), (3520, 2048, 512), (700, 1040, 1024), (1, 8192, 3072)])
def test_swiglu_large(m, h, k):
    check_swiglu(m, h, k, bias=m != 700)
    assert_no_device_error()


# ---------------------------------------------------------------- how they are called
def test_repeats_are_equal():
    """The same inputs give the same bits, whatever ran before."""
    from recavsr_b200.runtime import fp8_block
    for m, n, k in ((3, 3072, 2048), (200, 300, 1024), (1500, 1024, 512)):
        (ac, asc), (bc, bsc), _, _ = operands(m, n, k, 17)
        first = fp8_block.mm(ac, bc, asc, bsc)
        for _ in range(5):
            assert torch.equal(fp8_block.mm(ac, bc, asc, bsc), first)


def test_chain_without_syncs_on_another_stream():
    """Norm -> product -> quantize -> gated product queued back to back: each
    kernel starts while its predecessor ends and must read its finished output."""
    from recavsr_b200.runtime import fp8_block
    x, r = activations(333, 512, torch.bfloat16, 18), activations(333, 512, torch.bfloat16, 19)
    w = torch.ones(512, device="cuda")
    wq = fp8_block.quantize_weight(activations(512, 512, torch.bfloat16, 20))
    gu = fp8_block.quantize_weight(fp8_block.interleave_gate_up(*activations(1024, 512, torch.bfloat16, 21).chunk(2)))

    def chain():
        c, s, h = fp8_block.rms_norm_quantize(x, w, 1e-5, residual=r)
        o = fp8_block.mm(c, wq[0], s, wq[1], residual=h)
        c, s = fp8_block.quantize(o)
        return (*fp8_block.swiglu_mm(c, gu[0], s, gu[1]), o)

    want = chain()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [chain() for _ in range(20)]
    torch.cuda.synchronize()
    for g in got:
        for a, b in zip(g, want):
            assert torch.equal(a, b)


def test_graph_capture():
    from recavsr_b200.runtime import fp8_block
    (ac, asc), (bc, bsc), _, _ = operands(20, 256, 1024, 22)
    want = fp8_block.mm(ac, bc, asc, bsc)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = fp8_block.mm(ac, bc, asc, bsc)
    got.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_linear():
    from recavsr_b200.runtime import fp8_block
    torch.manual_seed(0)
    lin = torch.nn.Linear(528, 200, device="cuda", dtype=torch.bfloat16)
    q = fp8_block.BlockFP8Linear(lin)
    x = activations(6, 528, torch.bfloat16, 23).reshape(2, 3, 528)
    got, want = q(x).double(), lin(x).double()
    assert got.shape == (2, 3, 200) and q(x).dtype == torch.bfloat16
    # Each operand is rounded to 4 significant bits: relative errors up to 2^-4 of each of two factors, independent
    # over 528 terms, so the result's 2-norm is within 2^-4 sqrt(2 / 3) of the sum's (uniform rounding), under 6 %.
    assert float((got - want).detach().norm() / want.detach().norm()) < 0.06
    model = torch.nn.Sequential(lin, torch.nn.ReLU(), torch.nn.Linear(200, 16, bias=False, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="multiple of 16"):
        fp8_block.quantize_block_linears(model)     # 200 input features
    model = torch.nn.Sequential(lin, torch.nn.ReLU())
    fp8_block.quantize_block_linears(model)
    assert isinstance(model[0], fp8_block.BlockFP8Linear)


def test_linear_compiles():
    """torch.compile(fullgraph=True) traces through BlockFP8Linear."""
    from recavsr_b200.runtime import fp8_block
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(256, 512), torch.nn.GELU(), torch.nn.Linear(512, 128))
    model = model.to("cuda", torch.bfloat16)
    fp8_block.quantize_block_linears(model)
    x = activations(37, 256, torch.bfloat16, 24)
    with torch.inference_mode():
        want = model(x)
        got = torch.compile(model, fullgraph=True, backend="aot_eager")(x)
    assert torch.equal(got, want)


def test_refusals():
    from recavsr_b200.runtime import fp8_block
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    q, s = fp8_block.quantize(x)
    w = torch.ones(64, device="cuda")
    bad = [
        (lambda: fp8_block.quantize(x[:, :40]), "multiple of 16"),
        (lambda: fp8_block.quantize(x[0]), "2-D"),
        (lambda: fp8_block.quantize(x.to(torch.int32)), "float32 / bfloat16 / float16"),
        (lambda: fp8_block.rms_norm_quantize(x, w[:32], 1e-5), "weight"),
        (lambda: fp8_block.rms_norm_quantize(x, w, 1e-5, residual=x.float()), "residual"),
        (lambda: fp8_block.rms_norm_quantize(torch.zeros(1, 16400, device="cuda"), torch.ones(16400, device="cuda"),
                                             1e-5), "16384"),
        (lambda: fp8_block.mm(q, q[:, :48], s, s), "operands"),
        (lambda: fp8_block.mm(q, q, s[:256], s), "scale bytes"),
        (lambda: fp8_block.mm(q, q, s, s, w), "bias"),
        (lambda: fp8_block.mm(q, q, s, s, dtype=torch.float32), "bfloat16 or float16"),
        (lambda: fp8_block.mm(q, q, s, s, residual=x), "residual"),
        (lambda: fp8_block.mm(q, q, s, s, out=x), "out"),
        (lambda: fp8_block.mm(q.cpu(), q, s, s), "CUDA"),
        (lambda: fp8_block.swiglu_mm(q, q, s, s), "interleaved"),
    ]
    for call, words in bad:
        with pytest.raises(ValueError, match=words):
            call()
