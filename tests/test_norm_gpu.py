"""Residual addition + root-mean-square norm into the quantized activation
(qmm_rms_norm_act), such an activation read back (qmm_dequantize_act) and the
products from it (qmm_forward_act and its shared and GLU forms).

The normed values are held against 64 bits: rs, h * rs and * w each round once
in f32 (2^-24 relative each, eps / 2), and the sum of squares runs in 64 bits,
so y is within 3 * 2^-24 (1 + 2^-20) of the exact value. The planes are held to
QAct.quantize of the kernel's own f32 y, bit for bit (that quantizer is pinned
against the CPU oracle elsewhere), the stream to torch's rounding of the f32 sum.
"""
import pytest
import torch

from swarmllm_amd import GgmlDType, QAct, QMatMul, QTensor, fill_normal, forward_glu, rms_norm_act
from swarmllm_amd import _lib
from swarmllm_amd.qtensor import act_planes

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
EPS = 1e-5


def stream(rows, k, dtype, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(rows, k, generator=g, device="cuda")
    x[:, :: max(1, k // 7)] *= 20.0
    return x.to(dtype), torch.randn(rows, k, generator=g, device="cuda").to(dtype), \
        1.0 + 0.2 * torch.randn(k, generator=g, device="cuda")


def check_planes(act, y):
    want = QAct.quantize(y, GgmlDType.Q4K if act.layout == _lib.ACT_Q8K else GgmlDType.Q8_0)
    for got, ref in zip(act.planes(), want.planes()):
        assert torch.equal(got, ref)


def check_y(y, h, w, eps):
    h64 = h.double()
    want = h64 / (h64.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    assert (y.double() - want).abs().le(3 * 2.0**-24 * (1 + 2.0**-20) * want.abs() + 1e-45).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("weights", [GgmlDType.Q4K, GgmlDType.Q8_0])
@pytest.mark.parametrize("rows,k", [(1, 256), (3, 512), (5, 1024), (1, 1280), (2, 4096), (513, 1280), (600, 8192),
                                    (1, 8192), (7, 8448), (2, 16384), (1, 20480), (513, 20480), (1025, 256)])
def test_norm_quantize(dtype, weights, rows, k):
    x, r, w = stream(rows, k, dtype, rows + k)
    out = rms_norm_act(x, w, EPS, residual=r, dtype=weights, y_dtype=F32)
    assert torch.equal(out.h, (x.float() + r.float()).to(dtype))
    check_y(out.y, out.h, w, EPS)
    check_planes(out.act, out.y)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,k", [(1, 32), (4, 96), (9, 288), (1, 2880), (77, 2880), (600, 2880), (2, 4128),
                                    (3, 16416), (520, 8224)])
def test_norm_quantize_q8_0_ragged_k(dtype, rows, k):
    """Row lengths that end inside a wave's 256 values."""
    x, r, w = stream(rows, k, dtype, rows * 3 + k)
    out = rms_norm_act(x, w, EPS, residual=r, dtype=GgmlDType.Mxfp4, y_dtype=F32)
    assert torch.equal(out.h, (x.float() + r.float()).to(dtype))
    check_y(out.y, out.h, w, EPS)
    check_planes(out.act, out.y)


@pytest.mark.parametrize("k", [4, 100, 2884, 17000])
def test_norm_without_quantization(k):
    x, r, w = stream(5, k, F32, k)
    out = rms_norm_act(x, w, EPS, residual=r, dtype=None, y_dtype=F32)
    assert out.act is None
    check_y(out.y, out.h, w, EPS)
    # y in 16 bits: the f32 y rounded once
    for t in (F16, BF16):
        assert torch.equal(rms_norm_act(x, w, EPS, residual=r, dtype=None, y_dtype=t).y, out.y.to(t))


def test_a_row_does_not_depend_on_its_batch():
    """Every launch shape (rows from 1 to past 512) gives a row the same bits."""
    for k in (1280, 4096, 8192):
        x, r, w = stream(700, k, F32, k)
        whole = rms_norm_act(x, w, EPS, residual=r, y_dtype=F32)
        for i in (0, 1, 699):
            one = rms_norm_act(x[i:i + 1], w, EPS, residual=r[i:i + 1], y_dtype=F32)
            assert torch.equal(one.y[0], whole.y[i])
            for a, b in zip(one.act.planes(), whole.act.planes()):
                assert torch.equal(a[0], b[i])


def test_no_residual_and_in_place_streams():
    x, r, w = stream(6, 2048, F32, 3)
    plain = rms_norm_act(x, w, EPS, y_dtype=F32)
    assert plain.h is x
    check_y(plain.y, x, w, EPS)
    kept = torch.empty_like(x)
    assert rms_norm_act(x, w, EPS, h=kept).h is kept and torch.equal(kept, x)
    for big in (2048, 20480):
        x, r, w = stream(6, big, F32, 4)
        want = rms_norm_act(x, w, EPS, residual=r, y_dtype=F32)
        for which in ("x", "residual"):
            a, b = x.clone(), r.clone()
            got = rms_norm_act(a, w, EPS, residual=b, y_dtype=F32, h=a if which == "x" else b)
            assert torch.equal(got.y, want.y) and torch.equal(a if which == "x" else b, want.h)
            assert torch.equal(got.act.dequantize(), want.act.dequantize())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strided_and_unaligned_rows(dtype):
    x, r, w = stream(9, 3 * 512 + 5, dtype, 8)
    w = w[:512].contiguous()
    for off in (0, 4, 1, 515):
        xs, rs = x[:, off:off + 512], r[:, off:off + 512]
        got = rms_norm_act(xs, w, EPS, residual=rs, y_dtype=F32)
        want = rms_norm_act(xs.contiguous(), w, EPS, residual=rs.contiguous(), y_dtype=F32)
        assert torch.equal(got.h, want.h) and torch.equal(got.y, want.y)
        assert torch.equal(got.act.dequantize(), want.act.dequantize())
    # a three-dimensional stream keeps its shape
    y = rms_norm_act(x[:, :512].contiguous().view(3, 3, 512), w, EPS)
    assert y.act.shape == (3, 3, 512) and y.h.shape == (3, 3, 512)


def test_zero_tiny_and_non_finite_rows():
    x = torch.zeros(6, 1024, device="cuda")
    x[1] = 1e-30
    x[2] = 3e18  # squares past f32's range
    x[3, 5] = float("inf")
    x[4, 7] = float("nan")
    x[5] = 1e-42
    w = torch.ones(1024, device="cuda")
    for weights in (GgmlDType.Q4K, GgmlDType.Q8_0):
        out = rms_norm_act(x, w, EPS, dtype=weights, y_dtype=F32)
        check_y(out.y[:3], x[:3], w, EPS)
        assert (out.y[0] == 0).all() and torch.isnan(out.y[3, 5]) and torch.isnan(out.y[4]).all()
        check_planes(out.act, out.y)
    zero = rms_norm_act(x[:1], w, 0.0, y_dtype=F32)  # 0 / 0
    assert torch.isnan(zero.y).all()


@pytest.mark.parametrize("layout", [GgmlDType.Q6K, GgmlDType.Iq4Nl])
@pytest.mark.parametrize("rows,k", [(1, 256), (7, 2816), (65, 4096)])
def test_dequantize_act(layout, rows, k):
    x, _, _ = stream(rows, k, F32, k)
    act = QAct.quantize(x, layout)
    codes, scales, _ = act.planes()
    want = codes.float() * scales.repeat_interleave(k // scales.shape[1], 1)
    assert torch.equal(act.dequantize(), want)
    assert torch.equal(act.dequantize_f16(), want.half())
    assert torch.equal(act.dequantize(BF16), want.bfloat16())


@pytest.mark.parametrize("t", [GgmlDType.Q4K, GgmlDType.Q6K, GgmlDType.Q8_0, GgmlDType.Iq4Nl, GgmlDType.Mxfp4])
@pytest.mark.parametrize("rows", [1, 2, 3, 8, 21, 77, 130, 300])
@pytest.mark.parametrize("n,k", [(1024, 2048), (320, 4608)])
def test_products_from_the_planes(t, rows, n, k):
    """QMatMul.forward, forward_shared and forward_glu of a QAct give the bits
    of the f32 activation that it was quantized from."""
    ws = [QMatMul(QTensor.quantize(fill_normal(n * k, seed=s, std=0.02).reshape(n, k), t)) for s in (1, 2, 3)]
    x = fill_normal(rows * k, seed=9).reshape(rows, k)
    act = QAct.quantize(x, t)
    assert torch.equal(ws[0].forward(act), ws[0].forward(x))
    for a, b in zip(QMatMul.forward_shared(act, ws), QMatMul.forward_shared(x, ws)):
        assert torch.equal(a, b)
    assert torch.equal(forward_glu(act, ws[0], ws[1]), forward_glu(x, ws[0], ws[1]))


def test_products_from_the_planes_of_long_rows():
    """Rows past what the streaming kernel holds (1 row of more than 8192, 2 of more than 4096)."""
    for rows, n, k in ((1, 512, 8192), (1, 512, 11008), (2, 2048, 4096), (2, 512, 8192)):
        ws = [QMatMul(QTensor.quantize(fill_normal(n * k, seed=s, std=0.02).reshape(n, k), GgmlDType.Q4K)) for s in (1, 2)]
        x = fill_normal(rows * k, seed=9).reshape(rows, k)
        act = QAct.quantize(x, GgmlDType.Q4K)
        assert torch.equal(ws[0].forward(act), ws[0].forward(x))
        assert torch.equal(forward_glu(act, *ws), forward_glu(x, *ws))


def test_refusals():
    x, r, w = stream(4, 512, F32, 1)
    for bad in (lambda: rms_norm_act(x.cpu(), w, EPS), lambda: rms_norm_act(x.double(), w, EPS),
                lambda: rms_norm_act(x, w[:-1], EPS), lambda: rms_norm_act(x, w.half(), EPS),
                lambda: rms_norm_act(x, w, -1.0), lambda: rms_norm_act(x, w, float("nan")),
                lambda: rms_norm_act(x, w, EPS, residual=r[:3]), lambda: rms_norm_act(x, w, EPS, residual=r.half()),
                lambda: rms_norm_act(x, w, EPS, residual=r[:1].expand(4, 512)),
                lambda: rms_norm_act(x.t().contiguous().t(), w, EPS), lambda: rms_norm_act(x, w, EPS, dtype=None),
                lambda: rms_norm_act(x, w, EPS, dtype=GgmlDType.F16),
                lambda: rms_norm_act(x[:, :510], w[:510], EPS, dtype=None, y_dtype=F32),
                lambda: rms_norm_act(x[:, :300], w[:300], EPS), lambda: rms_norm_act(x, w, EPS, h=x[:2]),
                lambda: rms_norm_act(x, w, EPS, y_dtype=torch.float64), lambda: QAct.quantize(x.half(), GgmlDType.Q4K),
                lambda: QAct.quantize(x, GgmlDType.F32)):
        with pytest.raises(ValueError):
            bad()
    act = QAct.quantize(x, GgmlDType.Q4K)
    q8 = QMatMul(QTensor.quantize(fill_normal(64 * 512, seed=1).reshape(64, 512), GgmlDType.Q8_0))
    q4 = QMatMul(QTensor.quantize(fill_normal(64 * 256, seed=1).reshape(64, 256), GgmlDType.Q4K))
    for w_ in (q8, q4):  # another layout, another k
        with pytest.raises(ValueError):
            w_.forward(act)
        with pytest.raises(ValueError):
            QMatMul.forward_shared(act, [w_, w_])
        with pytest.raises(ValueError):
            forward_glu(act, w_, w_)
    assert rms_norm_act(x[:0], w, EPS).act.rows == 0
    assert q4.forward(QAct.alloc((0, 256), _lib.ACT_Q8K)).shape == (0, 64)
