"""GPU parity of the 4-bit operators against the 64-bit restatement (oracle/fp4_oracle.py).

Codes, block scales, row scales and the producers' hidden states are held to
every bit.  Products: with S = sum |va vb| (outer scales included), the fp32
accumulation of K products in groups of at most a block adds at most
(K / 16 + 16) 2^-23 S (one step per block and per alignment inside a group),
and the output rounding half a step, finfo.eps / 2 of the value.  The GELU
multiplies the first by at most 1.13 and adds the tanh instruction's 2^-11 of
|y| / 2; SwiGLU's sigmoid costs (2 + |g|) 2^-22 of the value (exponential and
quotient to 2 units each).
"""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import fp4_oracle as f4
from oracle import w8a8_oracle as orc

pytestmark = pytest.mark.gpu

FORMATS = ("nvfp4", "mxfp4")
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _check_quant(got, x, fmt, given=None):
    q, blocks, scales = got
    q_ref, b_ref, s_ref = f4.quantise(x.reshape(-1, x.shape[-1]), fmt, given)
    np.testing.assert_array_equal(blocks.view(torch.uint8).cpu().numpy(), b_ref)
    np.testing.assert_array_equal(q.cpu().numpy().reshape(q_ref.shape), q_ref)
    if fmt == "nvfp4" and given is None:
        np.testing.assert_array_equal(scales.cpu().numpy().reshape(-1), s_ref)
        assert scales.shape == (s_ref.size, 1)
    if fmt == "mxfp4":
        assert scales is None


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize(
    "rows,cols",
    [(1, 32), (3, 64), (7, 96), (33, 160), (130, 1376), (257, 2688), (5, 5376), (2, 12288),
     (1, 20000), (2, 33024)],
)
def test_quant_bit_exact(tm_ops, cuda, rows, cols, dtype, fmt):
    x = orc.activation(rows, cols, rows * 7919 + cols, outlier_channels=None).to(dtype)
    got = tm_ops.scaled_fp4_quant(x.to(cuda), block_format=fmt)
    assert got[0].shape == (rows, cols // 2) and got[0].dtype == torch.uint8
    assert got[1].dtype == (torch.float8_e4m3fn if fmt == "nvfp4" else torch.float8_e8m0fnu)
    _check_quant(got, x, fmt)


def _borders(dtype):
    """Rows whose elements sit on, just below and just above the code borders
    of scales with every mantissa, and rows of extremes."""
    rows = []
    for mantissa in range(8):
        s = 1.0 + mantissa / 8
        for top in (6.0, 5.0, 4.5, 5.25):  # 5.25 = 21 / 4: a row scale that is exact
            t = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
            step = torch.finfo(dtype).eps
            near = torch.cat((t, t * (1 + step), t * (1 - step)))
            row = torch.zeros(64, dtype=torch.float64)
            row[:21] = near * s
            row[21] = -top * s
            row[32:53] = -near * s * 0.5
            row[63] = 2.0 ** (mantissa - 4)
            rows.append(row)
    x = torch.stack(rows)
    x = torch.cat((x, x * 0.1, x * 448, x * (1 / 3)), 0)
    return x.to(dtype)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quant_on_the_borders(tm_ops, cuda, dtype, fmt):
    x = _borders(dtype)
    _check_quant(tm_ops.scaled_fp4_quant(x.to(cuda), block_format=fmt), x, fmt)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("given", [1.0, 1 / 3, 0.0371, 90.0 / 2688, 1000.0, 1e-5])
def test_quant_given_scale(tm_ops, cuda, dtype, given):
    x = torch.cat((_borders(dtype), orc.activation(9, 64, 3, outlier_channels=None).to(dtype)))
    scale = torch.tensor([given], device=cuda)
    got = tm_ops.scaled_fp4_quant(x.to(cuda), scale)
    assert got[2] is scale
    _check_quant(got, x, "nvfp4", given)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quant_extreme_rows(tm_ops, cuda, dtype, fmt):
    x = torch.randn(12, 512, generator=torch.Generator().manual_seed(1))
    x[0] = 0.0
    x[1] = -0.0
    x[2] *= 1e-40  # subnormal
    x[3] *= 1e-35
    x[4] *= 1e38
    x[5, 7] = float("inf")
    x[6, 100] = float("-inf")
    x[7, 511] = float("nan")
    x[8, :] = 0.0
    x[8, 5] = 3.0  # one block in use
    x[9, :16] *= 1e-6  # blocks whose scale underflows to 0
    x[10] = torch.finfo(dtype).max
    x[11] = torch.finfo(dtype).tiny
    x = x.to(dtype)
    got = tm_ops.scaled_fp4_quant(x.to(cuda), block_format=fmt)
    _check_quant(got, x, fmt)
    if fmt == "nvfp4":
        assert torch.isnan(got[2][5:8]).all()
        _check_quant(tm_ops.scaled_fp4_quant(x.to(cuda), torch.tensor([0.01], device=cuda)), x, fmt,
                     0.01)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quant_ties_under_every_row_maximum(tm_ops, cuda, dtype):
    """Every significand of a row maximum a (p bits), against elements that make
    x / (a / 2688 s) a border exactly, or miss one by a unit in the last place."""
    p = 8 if dtype == torch.bfloat16 else 11
    a = torch.arange(1 << (p - 1), 1 << p, dtype=torch.float64)
    if len(a) > 300:
        a = a[:: 7]
    t = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    s = torch.arange(8, 16, dtype=torch.float64)
    want = a.view(-1, 1, 1) / 2688 * s.view(1, -1, 1) * 16 * t.view(1, 1, -1)  # [a, s, t]
    x = torch.zeros(len(a), 8, 32, dtype=torch.float64)
    step = torch.finfo(dtype).eps
    x[:, :, 0:7], x[:, :, 7:14] = want, -want * (1 + step)
    x[:, :, 16:23], x[:, :, 23:30] = want * (1 - step), want
    # the element that gives the block its scale s: 6 s of the unit
    x[:, :, 14] = x[:, :, 30] = a.view(-1, 1) / 2688 * s * 16 * 6
    x = torch.cat((x.reshape(len(a), -1), torch.zeros(len(a), 32, dtype=torch.float64)), 1)
    x[:, -1] = a  # the row maximum
    x = x.to(dtype)
    _check_quant(tm_ops.scaled_fp4_quant(x.to(cuda)), x, "nvfp4")


@pytest.mark.parametrize("fmt", FORMATS)
def test_quant_strides_and_alignment(tm_ops, cuda, fmt):
    big = orc.activation(40, 1024, 6, outlier_channels=None).bfloat16().to(cuda)
    for view in (big[:, :512], big[:, 8:520], big[:, 16:528], big[3:, 1:129], big[::2, :96],
                 big.reshape(8, 5, 1024), big.t()[:, :32], big[:, ::2], big[:1, :64].expand(9, 64),
                 big.view(-1).as_strided((30, 64), (32, 1)), big[0, :96]):
        _check_quant(tm_ops.scaled_fp4_quant(view, block_format=fmt), view.cpu().contiguous(), fmt)
    f = big.float()
    for view in (f[:, 4:516], f[:, 1:65]):
        _check_quant(tm_ops.scaled_fp4_quant(view, block_format=fmt), view.cpu().contiguous(), fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quant_rows_behind_the_last_are_left(tm_ops, cuda, fmt):
    x = orc.activation(130, 96, 2, outlier_channels=None).bfloat16().to(cuda)
    q = torch.full((140, 48), 0xAB, dtype=torch.uint8, device=cuda)
    blocks = torch.empty_like(tm_ops.scaled_fp4_quant(x, block_format=fmt)[1])
    s = torch.full((140, 1), 7.0, device=cuda)
    torch.ops.taomate_w8a8.scaled_fp4_quant(q[:130], blocks, s[:130] if fmt == "nvfp4" else None, x,
                                            None)
    assert (q[130:] == 0xAB).all() and (s[130:] == 7.0).all()
    empty = tm_ops.scaled_fp4_quant(x[:0], block_format=fmt)
    assert empty[0].shape == (0, 48) and empty[1].numel() == 0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,cols", [(1, 32), (130, 1376), (3, 20000)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_dequantise(tm_ops, cuda, rows, cols, out_dtype, fmt):
    x = orc.activation(rows, cols, rows + cols, outlier_channels=None).bfloat16()
    q, b, s = tm_ops.scaled_fp4_quant(x.to(cuda), block_format=fmt)
    got = tm_ops.dequantize_fp4(q, b, s, out_dtype).cpu().double().numpy()
    ref = f4.stored_values(q.cpu().numpy(), b.view(torch.uint8).cpu().numpy(), fmt)
    if s is not None:
        ref = ref * s.cpu().double().numpy()
    # one fp32 rounding of the product with the row scale, one to the output
    tol = np.abs(ref) * (HALF_STEP[out_dtype] + 2.0 ** -24) * (1 + 2.0 ** -8)
    if out_dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half a subnormal step
    assert (np.abs(got - ref) <= tol).all()


def test_dequantise_given_scale_and_nan(tm_ops, cuda):
    x = torch.randn(4, 64, generator=torch.Generator().manual_seed(3))
    x[1, 3] = float("nan")
    x[2, 40] = float("inf")
    scale = torch.tensor([0.01], device=cuda)
    y = tm_ops.dequantize_fp4(*tm_ops.scaled_fp4_quant(x.to(cuda), scale))
    assert torch.isnan(y[1, :16]).all() and torch.isfinite(y[1, 16:]).all()
    assert torch.isnan(y[2, 32:48]).all() and torch.isfinite(y[2, :32]).all()
    y = tm_ops.dequantize_fp4(*tm_ops.scaled_fp4_quant(x.to(cuda)))
    assert torch.isnan(y[1:3]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[3]).all()
    y = tm_ops.dequantize_fp4(*tm_ops.scaled_fp4_quant(x.to(cuda), block_format="mxfp4"))
    assert torch.isnan(y[1, :32]).all() and torch.isfinite(y[1, 32:]).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,cols,tables", [(1, 32, 0), (130, 1376, 3), (37, 3072, 0), (5, 5376, 2),
                                              (2, 20480, 1)])
@pytest.mark.parametrize("mode", ["modulate", "rms", "residual"])
def test_producers(tm_ops, cuda, mode, rows, cols, tables, fmt):
    """The hidden state and residual are the int8 producers' bits, and the
    codes those of the plain quantisation of that hidden state."""
    g = torch.Generator().manual_seed(rows + cols)
    rnd = lambda *shape, std=1.0: (torch.randn(shape, generator=g) * std).bfloat16().to(cuda)  # noqa: E731
    x, branch = rnd(rows, cols), rnd(rows, cols)
    shift, scale, gate = (rnd(tables or rows, cols, std=0.3) for _ in range(3))
    index = torch.randint(0, tables, (rows,), generator=g).to(cuda) if tables else None
    w = rnd(cols)
    if mode == "modulate":
        *got, hidden = tm_ops.modulate_fp4_quant(x, shift, scale, index, block_format=fmt,
                                                 return_hidden=True)
        ref = tm_ops.modulate_int8_quant(x, shift, scale, index, return_hidden=True)[-1]
    elif mode == "rms":
        *got, hidden = tm_ops.rms_norm_modulate_fp4_quant(x, w, 1e-6, shift, scale, index,
                                                          block_format=fmt, return_hidden=True)
        ref = tm_ops.rms_norm_modulate_int8_quant(x, w, 1e-6, shift, scale, index,
                                                  return_hidden=True)[-1]
    else:
        *got, res, hidden = tm_ops.residual_gate_rms_norm_modulate_fp4_quant(
            x, branch, gate, w, 1e-6, shift, scale, index, block_format=fmt, return_hidden=True)
        _, _, res_ref, ref = tm_ops.residual_gate_rms_norm_modulate_int8_quant(
            x, branch, gate, w, 1e-6, shift, scale, index, return_hidden=True)
        assert torch.equal(res, res_ref)
    assert torch.equal(hidden, ref)
    _check_quant(got, hidden.cpu(), fmt)
    if mode == "modulate":  # without the hidden state
        again = tm_ops.modulate_fp4_quant(x, shift, scale, index, block_format=fmt)
        assert again[3] is None and torch.equal(again[0], got[0])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("mode", ["modulate", "rms", "residual"])
def test_producers_tables_at_16_bytes(tm_ops, cuda, mode, shared, fmt):
    """Tables that are column slices of a larger tensor, their rows at 16 bytes
    off a multiple of 32, give the bits of contiguous ones."""
    rows, cols = 133, 1376
    g = torch.Generator().manual_seed(5)
    rnd = lambda *shape: torch.randn(shape, generator=g).bfloat16().to(cuda)  # noqa: E731
    x, branch, w = rnd(rows, cols), rnd(rows, cols), rnd(cols)
    sliced = [rnd(4 if shared else rows, cols + 24)[:, 8:cols + 8] for _ in range(3)]
    index = torch.randint(0, 4, (rows,), generator=g).to(cuda) if shared else None

    def run(shift, scale, gate):
        if mode == "modulate":
            return tm_ops.modulate_fp4_quant(x, shift, scale, index, block_format=fmt,
                                             return_hidden=True)
        if mode == "rms":
            return tm_ops.rms_norm_modulate_fp4_quant(x, w, 1e-6, shift, scale, index,
                                                      block_format=fmt, return_hidden=True)
        return tm_ops.residual_gate_rms_norm_modulate_fp4_quant(
            x, branch, gate, w, 1e-6, shift, scale, index, block_format=fmt, return_hidden=True)

    for a, b in zip(run(*sliced), run(*(t.contiguous() for t in sliced)), strict=True):
        assert (a is None and b is None) or torch.equal(a, b)


# ---------------------------------------------------------------- product
def _operands(tm_ops, cuda, m, n, k, fmt, dtype, seed):
    x = orc.activation(m, k, seed, outlier_channels=None).bfloat16().to(cuda)
    w = orc.weight(n, k, seed=seed + 1).to(cuda)
    g = torch.Generator().manual_seed(seed + 2)
    bias = (torch.randn(n, generator=g) * 0.3).to(dtype).to(cuda)
    return (*tm_ops.scaled_fp4_quant(x, block_format=fmt),
            *tm_ops.scaled_fp4_quant(w, block_format=fmt), bias)


def _values(q, b, s, fmt):
    v = f4.stored_values(q.cpu().numpy(), b.view(torch.uint8).cpu().numpy(), fmt)
    return v if s is None else v * s.cpu().double().numpy().reshape(-1, 1)


def _check_mm(out, aq, ab, asc, wq, wb, wsc, bias, fmt, act="none"):
    a, b = (torch.from_numpy(_values(*t, fmt)).to(out.device) for t in ((aq, ab, asc), (wq, wb, wsc)))
    k = a.shape[1]
    y = (a @ b.t()).cpu().numpy()
    size = (a.abs() @ b.abs().t()).cpu().numpy()
    slack = (k / 16 + 16) * 2.0 ** -23 * size
    if bias is not None:
        y = y + bias.cpu().double().numpy()
        slack = slack + 2.0 ** -23 * np.abs(y)
    half = HALF_STEP[out.dtype]
    if act == "gelu":
        ref = f4.gelu_tanh(y)
        tol = 1.13 * slack + np.abs(y) / 2 * 2.0 ** -11
    elif act == "swiglu":
        ref = f4.swiglu(y)
        p, s = y.reshape(y.shape[0], -1, 2, 16), slack.reshape(y.shape[0], -1, 2, 16)
        g, u = p[:, :, 0], p[:, :, 1]
        # d(g sigmoid(g)) <= 1.1 dg; |g sigmoid(g)| <= |g|
        tol = (1.1 * s[:, :, 0] * (np.abs(u) + s[:, :, 1]) + np.abs(g) * s[:, :, 1]).reshape(ref.shape)
        tol = tol + np.abs(ref) * (2 + np.abs(g).reshape(ref.shape)) * 2.0 ** -22
    else:
        ref, tol = y, slack
    tol = tol + half * (np.abs(ref) + tol)
    if out.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    err = np.abs(out.cpu().double().numpy() - ref)
    assert (err <= tol).all(), (float((err / tol).max()), np.argwhere(err > tol)[:4], err.max())


SMALL = [(32, 1), (32, 2), (32, 4), (32, 8), (64, 1), (64, 4), (128, 1), (128, 2), (128, 8)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tile,splits", SMALL)
@pytest.mark.parametrize("m,n,k", [(1, 128, 2048), (31, 200, 2336), (17, 8, 2592), (32, 1160, 2048 + 96)])
def test_mm_small_tiles(tm_ops, cuda, m, n, k, tile, splits, fmt):
    *ops, bias = _operands(tm_ops, cuda, m, n, k, fmt, torch.bfloat16, m + n + k)
    aq, ab, asc, wq, wb, wsc = ops
    out = tm_ops.scaled_mm_fp4(aq, wq.t(), ab, wb, asc, wsc, bias=bias, tile=tile, splits=splits)
    _check_mm(out, *ops, bias, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k", [32, 64, 96, 128, 160, 224, 256, 288, 512, 1376])
def test_mm_every_k_tail(tm_ops, cuda, k, dtype, fmt):
    *ops, bias = _operands(tm_ops, cuda, 70, 136, k, fmt, dtype, k)
    aq, ab, asc, wq, wb, wsc = ops
    _check_mm(tm_ops.scaled_mm_fp4(aq, wq.t(), ab, wb, asc, wsc, dtype), *ops, None, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("act", ["none", "gelu", "swiglu"])
@pytest.mark.parametrize("m,n,k", [(1, 64, 256), (60, 704, 1024), (300, 1344, 800), (1003, 1152, 1376)])
def test_mm_epilogues(tm_ops, cuda, m, n, k, act, fmt):
    *ops, bias = _operands(tm_ops, cuda, m, n, k, fmt, torch.bfloat16, m + n)
    aq, ab, asc, wq, wb, wsc = ops
    for b in (None, bias):
        out = tm_ops.scaled_mm_fp4(aq, wq.t(), ab, wb, asc, wsc, bias=b, gelu_tanh=act == "gelu",
                                   swiglu=act == "swiglu")
        _check_mm(out, *ops, b, fmt, act)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("act,dtype", [("none", torch.bfloat16), ("gelu", torch.float16),
                                       ("swiglu", torch.bfloat16)])
@pytest.mark.parametrize("m,n,k", [(1, 64, 32), (256, 256, 256), (129, 448, 96), (300, 1344, 800),
                                   (517, 2112, 1376), (2049, 5120, 544), (5000, 4160, 288)])
def test_mm_pair_tile(tm_ops, cuda, m, n, k, act, dtype, fmt):
    """The CTA-pair kernel: one tile to several waves, tails in every dimension."""
    *ops, bias = _operands(tm_ops, cuda, m, n, k, fmt, dtype, m + n + k)
    aq, ab, asc, wq, wb, wsc = ops
    out = tm_ops.scaled_mm_fp4(aq, wq.t(), ab, wb, asc, wsc, dtype, bias, gelu_tanh=act == "gelu",
                               swiglu=act == "swiglu", tile=1256)
    _check_mm(out, *ops, bias, fmt, act)
    plain = tm_ops.scaled_mm_fp4(aq, wq.t(), ab, wb, asc, wsc, dtype, tile=1256)
    _check_mm(plain, *ops, None, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 2, 33, 64, 65, 128, 129, 700])
def test_mm_every_route(tm_ops, cuda, m, fmt):
    """The chosen kernel at the token counts where the choice changes, long K."""
    *ops, bias = _operands(tm_ops, cuda, m, 520, 5376, fmt, torch.bfloat16, m)
    aq, ab, asc, wq, wb, wsc = ops
    _check_mm(tm_ops.scaled_mm_fp4(aq, wq.t(), ab, wb, asc, wsc, bias=bias), *ops, bias, fmt)


def _slots(n, offset, dtype, cuda, fill=0.0):
    """n values that start `offset` elements into their storage."""
    return torch.full((n + offset,), fill, dtype=dtype, device=cuda)[offset:]


@pytest.mark.parametrize("tile", [0, 64, 1256])
@pytest.mark.parametrize("fmt", FORMATS)
def test_mm_strides_and_alignment(tm_ops, cuda, fmt, tile):
    """Row-strided codes and output, scales and bias at odd addresses; what lies
    beside the output stays as it was."""
    m, n, k = 60, 392, 672
    *ops, bias = _operands(tm_ops, cuda, m, n, k, fmt, torch.bfloat16, 5)
    aq, ab, asc, wq, wb, wsc = ops
    a_big = torch.randint(0, 255, (m, k // 2 + 48), dtype=torch.uint8, device=cuda)
    w_big = torch.randint(0, 255, (n, k // 2 + 16), dtype=torch.uint8, device=cuda)
    a_big[:, 16:16 + k // 2] = aq
    w_big[:, :k // 2] = wq
    if wsc is not None:
        asc, wsc = _slots(m, 1, torch.float32, cuda).copy_(asc.view(-1)), \
            _slots(n, 3, torch.float32, cuda).copy_(wsc.view(-1))
    bias = _slots(n, 1, torch.bfloat16, cuda).copy_(bias)
    for width, start in ((n + 8, 8), (n + 24, 16)):  # rows on 16- and on 32-byte boundaries
        big = torch.full((m + 2, width), 7.0, dtype=torch.bfloat16, device=cuda)
        out = big[1:m + 1, start:start + n]
        if out.data_ptr() % 16:
            continue
        torch.ops.taomate_w8a8.scaled_mm_fp4(
            out, a_big[:, 16:16 + k // 2], w_big[:, :k // 2].t(), ab, wb, asc, wsc, bias, 0, tile, 1)
        _check_mm(out, aq, ab, asc, wq, wb, wsc, bias, fmt)
        keep = torch.ones_like(big, dtype=torch.bool)
        keep[1:m + 1, start:start + n] = False
        assert (big[keep] == 7.0).all()


@pytest.mark.parametrize("tile,splits", [(32, 1), (32, 4), (128, 2), (1256, 1)])
def test_mm_scalar_scales_and_shapes(tm_ops, cuda, tile, splits):
    """Per-tensor scales on either side, a given activation scale, 3-D input, `out`."""
    m, n, k = 24, 136, 1024
    x = orc.activation(m, k, 1, outlier_channels=None).bfloat16().to(cuda)
    w = orc.weight(n, k, seed=2).to(cuda)
    sx, sw = torch.tensor([0.002], device=cuda), torch.tensor([0.0001], device=cuda)
    aq, ab, asc = tm_ops.scaled_fp4_quant(x, sx)
    wq, wb, wsc = tm_ops.scaled_fp4_quant(w, sw)
    out = torch.empty(m, n, dtype=torch.float16, device=cuda)
    got = tm_ops.scaled_mm_fp4(aq, wq.t(), ab, wb, asc, wsc, out=out, tile=tile, splits=splits)
    assert got is out
    _check_mm(out, aq, ab, asc, wq, wb, wsc, None, "nvfp4")
    q3, b3, s3 = tm_ops.scaled_fp4_quant(x.view(2, 12, k))
    assert q3.shape == (2, 12, k // 2) and s3.shape == (m, 1)
    y3 = tm_ops.scaled_mm_fp4(q3, wq.t(), b3, wb, s3, wsc)
    assert y3.shape == (2, 12, n)
    _check_mm(y3.view(m, n), q3.view(m, -1), b3, s3, wq, wb, wsc, None, "nvfp4")
    assert tm_ops.scaled_mm_fp4(aq[:0], wq.t(), *tm_ops.scaled_fp4_quant(x[:0])[1:2], wb,
                                asc, wsc).shape == (0, n)


@pytest.mark.parametrize("tile", [32, 1256])
@pytest.mark.parametrize("fmt", FORMATS)
def test_mm_nan_rows(tm_ops, cuda, fmt, tile):
    """An inf or NaN in a token makes its outputs NaN, in a weight row its
    column's, and nothing else."""
    x = orc.activation(20, 512, 1, outlier_channels=None).bfloat16()
    w = orc.weight(72, 512, seed=2).clone()
    x[3, 100], x[17, 511], w[40, 7] = float("nan"), float("inf"), float("-inf")
    x[5] = 0.0
    a, b = (tm_ops.scaled_fp4_quant(t.to(cuda), block_format=fmt) for t in (x, w))
    y = tm_ops.scaled_mm_fp4(a[0], b[0].t(), a[1], b[1], a[2], b[2], tile=tile).cpu()
    bad = torch.zeros(20, 72, dtype=torch.bool)
    bad[3], bad[17], bad[:, 40] = True, True, True
    assert torch.equal(torch.isnan(y), bad)
    assert (y[5][~bad[5]] == 0).all()


def test_streams_and_graphs(tm_ops, cuda):
    """Two streams at once, and two captured graphs replayed on new inputs while
    eager calls run: the calls share no scratch memory."""
    shapes = [(1, 1024, 4096), (48, 640, 5376), (300, 1344, 800), (2100, 4160, 544)]
    cases = []
    for m, n, k in shapes:
        x = orc.activation(m, k, m, outlier_channels=None).bfloat16().to(cuda)
        w = tm_ops.scaled_fp4_quant(orc.weight(n, k, seed=n).to(cuda))
        cases.append((x, w))

    def linear(x, w):
        q, b, s = tm_ops.scaled_fp4_quant(x)
        return tm_ops.scaled_mm_fp4(q, w[0].t(), b, w[1], s, w[2], gelu_tanh=True)

    want = [linear(x, w) for x, w in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = [linear(x, w) for x, w in (cases if i else cases[::-1])]
    torch.cuda.synchronize()
    for a, b, c in zip(want, got[1], got[0][::-1]):
        assert torch.equal(a, b) and torch.equal(a, c)

    graphs, outs = [], []
    inputs = [x.clone() for x, _ in cases]
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([linear(x, w) for x, (_, w) in zip(inputs, cases)])
        graphs.append(g)
    for x in inputs:
        x.mul_(0.5).neg_()
    torch.cuda.synchronize()
    for i, g in enumerate(graphs):
        with torch.cuda.stream(streams[i]):
            g.replay()
    eager = [linear(x, w) for x, (_, w) in zip(inputs, cases)]
    torch.cuda.synchronize()
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for o in outs:
        for a, b in zip(o, eager):
            assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", FORMATS)
def test_positions_past_32_bits(tm_ops, cuda, fmt):
    """More than 2^31 elements on either side of the quantisation, and an output of
    more than 2^31 elements: the far rows equal those of small calls."""
    rows, cols = 70_000, 32_768  # 2.3e9 elements
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=cuda)
    tail = orc.activation(130, cols, 3, outlier_channels=None).bfloat16().to(cuda)
    x[-130:] = tail
    q, b, s = tm_ops.scaled_fp4_quant(x, block_format=fmt)
    qt, _, st = tm_ops.scaled_fp4_quant(tail, block_format=fmt)
    assert torch.equal(q[-130:], qt) and (s is None or torch.equal(s[-130:], st))
    y = tm_ops.dequantize_fp4(q, b, s)
    assert torch.equal(y[-130:], tm_ops.dequantize_fp4(*tm_ops.scaled_fp4_quant(tail, block_format=fmt)))
    assert not y[:1000].any()
    del x, y
    w = tm_ops.scaled_fp4_quant(orc.weight(34_000, 64, seed=1).to(cuda), block_format=fmt)
    a = tm_ops.scaled_fp4_quant(orc.activation(rows, 64, 2, outlier_channels=None).bfloat16().to(cuda),
                                block_format=fmt)
    out = tm_ops.scaled_mm_fp4(a[0], w[0].t(), a[1], w[1], a[2], w[2])  # 2.4e9 outputs
    last = a[0][-100:].contiguous()
    va = _values(*a, fmt)[-100:]
    ref = va @ _values(*w, fmt).T
    size = np.abs(va) @ np.abs(_values(*w, fmt)).T
    err = np.abs(out[-100:].cpu().double().numpy() - ref)
    assert last.shape == (100, 32)
    assert (err <= 2.0 ** -8 * np.abs(ref) + (64 / 16 + 16) * 2.0 ** -22 * size).all()


def test_c_abi_linear(tm_ops, capi, cuda):
    """Quantisation, product and inverse through the C ABI alone."""
    m, n, k = 70, 200, 416
    x = orc.activation(m, k, 1, outlier_channels=None).bfloat16().to(cuda)
    w = orc.weight(n, k, seed=2).to(cuda)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for code, fmt in ((0, "nvfp4"), (1, "mxfp4")):
        parts = []
        for t, rows, dt in ((x, m, 0), (w, n, {torch.bfloat16: 0, torch.float32: 2}[w.dtype])):
            size = ctypes.c_uint64()
            assert capi.tm_fp4_block_scales_size(rows, k, code, ctypes.byref(size)) == 0
            q = torch.empty(rows, k // 2, dtype=torch.uint8, device=cuda)
            blocks = torch.empty(size.value, dtype=torch.uint8, device=cuda)
            s = torch.empty(rows, device=cuda) if code == 0 else None
            assert capi.tm_scaled_fp4_quant(q.data_ptr(), blocks.data_ptr(),
                                            None if s is None else s.data_ptr(), None, t.data_ptr(),
                                            dt, code, rows, k, k, stream) == 0
            ref = tm_ops.scaled_fp4_quant(t, block_format=fmt)
            assert torch.equal(q, ref[0]) and torch.equal(blocks, ref[1].view(torch.uint8).view(-1))
            back = torch.empty(rows, k, dtype=torch.float32, device=cuda)
            assert capi.tm_dequantize_fp4(back.data_ptr(), 2, q.data_ptr(), blocks.data_ptr(),
                                          None if s is None else s.data_ptr(), rows if s is not None else 0,
                                          code, rows, k, stream) == 0
            assert torch.equal(back, tm_ops.dequantize_fp4(*ref, torch.float32))
            parts.append((q, blocks, s))
        (aq, ab, sa), (wq, wb, sw) = parts
        out = torch.empty(m, n, dtype=torch.bfloat16, device=cuda)
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        assert capi.tm_scaled_mm_fp4(ptr(out), 0, ptr(aq), ptr(wq), ptr(ab), ptr(wb), ptr(sa),
                                     m if sa is not None else 0, ptr(sw), n if sw is not None else 0,
                                     None, code, m, n, k, k // 2, k // 2, n, 0, stream) == 0
        kind = torch.float8_e4m3fn if code == 0 else torch.float8_e8m0fnu
        shape = f4.scale_tiles(m, k, fmt), f4.scale_tiles(n, k, fmt)
        _check_mm(out, aq, ab.view(shape[0]).view(kind), sa, wq, wb.view(shape[1]).view(kind), sw,
                  None, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_block_run(tm_ops, cuda, fmt):
    """A block's MLP as it is used: gated residual + RMSNorm + modulate producer,
    fc1 with bias and GELU, quantisation, fc2.  Each product is held to the
    64-bit value of its own stored operands, each quantisation to every bit."""
    tokens, d, ffn = 333, 512, 1408
    g = torch.Generator().manual_seed(4)
    rnd = lambda *shape, std=1.0: (torch.randn(shape, generator=g) * std).bfloat16().to(cuda)  # noqa: E731
    residual, branch, weight = rnd(tokens, d), rnd(tokens, d), 1 + rnd(d, std=0.1)
    shift, scale, gate = (rnd(3, d, std=0.3) for _ in range(3))
    index = torch.randint(0, 3, (tokens,), generator=g).to(cuda)
    w1 = tm_ops.scaled_fp4_quant(rnd(ffn, d, std=0.05), block_format=fmt)
    w2 = tm_ops.scaled_fp4_quant(rnd(d, ffn, std=0.05), block_format=fmt)
    b1, b2 = rnd(ffn, std=0.2), rnd(d, std=0.2)
    q, b, s, new_residual, hidden = tm_ops.residual_gate_rms_norm_modulate_fp4_quant(
        residual, branch, gate, weight, 1e-6, shift, scale, index, block_format=fmt,
        return_hidden=True)
    _check_quant((q, b, s), hidden.cpu(), fmt)
    h = tm_ops.scaled_mm_fp4(q, w1[0].t(), b, w1[1], s, w1[2], bias=b1, gelu_tanh=True)
    _check_mm(h, q, b, s, *w1, b1, fmt, "gelu")
    q2, bb2, s2 = tm_ops.scaled_fp4_quant(h, block_format=fmt)
    _check_quant((q2, bb2, s2), h.cpu(), fmt)
    y = tm_ops.scaled_mm_fp4(q2, w2[0].t(), bb2, w2[1], s2, w2[2], bias=b2)
    _check_mm(y, q2, bb2, s2, *w2, b2, fmt)
    assert torch.isfinite(y).all() and new_residual.shape == residual.shape


@pytest.mark.parametrize("fmt", FORMATS)
def test_dit_mlp_stage(tm_ops, cuda, fmt):
    """dit.TPW4A4MLP is the operators in sequence, and can be captured."""
    from taomate_hd_b200.dit import TPW4A4MLP
    from taomate_hd_b200.parallel import ParallelContext

    ctx = ParallelContext(tp_world_size=1, tp_rank=0, tp_group=None)
    mlp = TPW4A4MLP(320, 256, 1024, ctx, cuda, seed=3, block_format=fmt)
    x = orc.activation(320, 256, 7, outlier_channels=1).bfloat16().to(cuda)
    got = mlp.forward(x).clone()
    q, b, s = tm_ops.scaled_fp4_quant(x, block_format=fmt)
    h = tm_ops.scaled_mm_fp4(q, mlp.fc1.q.t(), b, mlp.fc1.blocks, s, mlp.fc1.scale,
                             bias=mlp.fc1.bias, gelu_tanh=True)
    q, b, s = tm_ops.scaled_fp4_quant(h, block_format=fmt)
    want = tm_ops.scaled_mm_fp4(q, mlp.fc2.q.t(), b, mlp.fc2.blocks, s, mlp.fc2.scale,
                                bias=mlp.fc2.bias)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mlp.forward(x)
    x.mul_(2.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, mlp.forward(x)) and not torch.equal(out, got)


def test_refusals_on_device_tensors(tm_ops, cuda):
    """Wrong types, shapes and formats raise before any launch."""
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=cuda)
    q, b, s = tm_ops.scaled_fp4_quant(x)
    qm, bm, _ = tm_ops.scaled_fp4_quant(x, block_format="mxfp4")
    one = torch.ones(1, device=cuda)
    mm = tm_ops.scaled_mm_fp4
    w = torch.zeros(8, 64, dtype=torch.bfloat16, device=cuda)
    wq, wb, ws = tm_ops.scaled_fp4_quant(w)
    bad = [
        (lambda: tm_ops.scaled_fp4_quant(x.to(torch.int32)), RuntimeError),
        (lambda: tm_ops.scaled_fp4_quant(x[:, :48]), RuntimeError),
        (lambda: tm_ops.scaled_fp4_quant(x, one, block_format="mxfp4"), RuntimeError),
        (lambda: tm_ops.scaled_fp4_quant(x, torch.ones(4, device=cuda)), RuntimeError),
        (lambda: tm_ops.scaled_fp4_quant(x, block_format="fp4"), ValueError),
        (lambda: tm_ops.dequantize_fp4(q, b), RuntimeError),           # nvfp4 needs its scales
        (lambda: tm_ops.dequantize_fp4(qm, bm, one), RuntimeError),    # mxfp4 takes none
        (lambda: tm_ops.dequantize_fp4(q, b[:, :0], s), RuntimeError),
        (lambda: tm_ops.dequantize_fp4(q, b.view(torch.uint8), s), RuntimeError),
        (lambda: tm_ops.dequantize_fp4(q, b, s, torch.int8), RuntimeError),
        (lambda: mm(q, wq.t(), b, wb, s), RuntimeError),
        (lambda: mm(q, wq.t(), b, bm, s, ws), RuntimeError),           # two formats
        (lambda: mm(q, wq, b, wb, s, ws), RuntimeError),               # weight not transposed
        (lambda: mm(q, wq.t(), b, wb, s, ws, torch.float32), RuntimeError),
        (lambda: mm(q, wq.t(), b, wb, s, ws, bias=torch.zeros(8, device=cuda)), RuntimeError),
        (lambda: mm(q, wq.t(), b, wb, s, ws, swiglu=True), RuntimeError),  # N % 64
        (lambda: mm(q, wq.t(), b, wb, s, ws, gelu_tanh=True, swiglu=True), ValueError),
        (lambda: mm(q, wq.t(), b, wb, s, ws, tile=48), RuntimeError),
        (lambda: mm(q, wq.t(), b, wb, s, ws, tile=32, splits=2), RuntimeError),  # one k-block
        (lambda: mm(q, wq.t(), b, wb, s, ws, out=torch.empty(4, 4, device=cuda)), RuntimeError),
        (lambda: tm_ops.modulate_fp4_quant(x.float(), x[:1], x[:1], None), RuntimeError),
    ]
    for call, error in bad:
        with pytest.raises(error):
            call()


@pytest.mark.parametrize("tile", [32, 64, 128, 1256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_mm_gelu_is_rounded_once(tm_ops, cuda, dtype, tile):
    """GELU of exactly known arguments (zero products, so the bias), the negative
    ones among them, where 1 + tanh cancels.  With t = |2 u| / ln 2 the exponent
    of exp(-2 u) carries four roundings and the constants' (2^-22 t), the
    exponential and the reciprocal 2^-22 and 2^-23 (their documented bounds), the
    sum and the last product 2^-24 each: (t + 2) 2^-22 of the value, and the
    output's half step."""
    n = 2048
    y = torch.linspace(-9.0, 9.0, n, dtype=torch.float64)
    y[:8] = torch.tensor([-60.0, -20.0, 20.0, 60.0, 0.0, -0.0, -5.5, 1e-3])
    bias = y.to(dtype)
    x = tm_ops.scaled_fp4_quant(torch.zeros(5, 64, dtype=dtype, device=cuda))
    w = tm_ops.scaled_fp4_quant(orc.weight(n, 64, seed=2).to(cuda))
    out = tm_ops.scaled_mm_fp4(x[0], w[0].t(), x[1], w[1], x[2], w[2], dtype, bias.to(cuda),
                               gelu_tanh=True, tile=tile).cpu().double()
    y = bias.double()
    two_u = 2.0 * (2.0 / torch.pi) ** 0.5 * (y + 0.044715 * y ** 3)
    ref = y / (1.0 + torch.exp(-two_u))
    t = two_u.abs() / 0.6931
    tol = ref.abs() * (HALF_STEP[dtype] * (1 + 2.0 ** -10) + (t + 2) * 2.0 ** -22)
    tol = tol + y.abs() * 2.0 ** -126 + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134)
    assert ((out - ref).abs() <= tol).all(), ((out - ref).abs() / tol).max()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-6])
@pytest.mark.parametrize("rows,cols,tables", [(20, 32, 0), (20, 1376, 3), (20, 5376, 0), (20, 20480, 2)])
@pytest.mark.parametrize("mode", ["rms", "residual"])
def test_norm_of_extreme_rows(tm_ops, cuda, mode, rows, cols, tables, eps, fmt):
    """Rows whose squares leave the range of fp32, beside ordinary ones, against the
    norm in 64 bits.  Shift and scale are 0, so the hidden state is
    bf16(x rinv w): rinv carries four fp32 roundings (mean, eps, root, reciprocal),
    the products two more, 6 2^-24 < 2^-21 of the value; then half a bf16 step, 2^-8.
    Scaled rows lose at most 2^-134 times 1 / rms <= 2 in their subnormals, and the
    output as much again: 2^-132."""
    g = torch.Generator().manual_seed(cols)
    x = torch.randn((rows, cols), generator=g)
    power = torch.tensor([0, 60, 62, 63, 64, 70, 100, 120, 125, 0, -30, -40, -45, -50, -60, -64, -70,
                          -100, -120, -128])
    x = torch.ldexp(x.clamp(-3.9, 3.9), power.view(-1, 1)).bfloat16()
    x[9, 1:] *= 2.0 ** -100  # one value carries the row
    w = (1 + 0.1 * torch.randn(cols, generator=g)).bfloat16()
    table = torch.zeros(tables or rows, cols, dtype=torch.bfloat16, device=cuda)
    index = (torch.arange(rows, device=cuda) % tables) if tables else None
    if mode == "rms":
        *got, hidden = tm_ops.rms_norm_modulate_fp4_quant(
            x.to(cuda), w.to(cuda), eps, table, table, index, block_format=fmt, return_hidden=True)
    else:
        *got, residual, hidden = tm_ops.residual_gate_rms_norm_modulate_fp4_quant(
            x.to(cuda), torch.ones_like(x, device=cuda), table, w.to(cuda), eps, table, table, index,
            block_format=fmt, return_hidden=True)
        assert torch.equal(residual.cpu(), x)
    _check_quant(got, hidden.cpu(), fmt)
    v = x.double()
    eps = torch.tensor(eps, dtype=torch.float32).double()
    ref = v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps) * w.double()
    err = (hidden.cpu().double() - ref).abs()
    tol = ref.abs() * (2.0 ** -8 + 2.0 ** -21) + 2.0 ** -132
    assert (err <= tol).all(), (err / tol).amax(-1)


@pytest.mark.parametrize("fmt", FORMATS)
def test_norm_of_rows_without_a_value(tm_ops, cuda, fmt):
    """An infinity or a NaN beside huge rows: its row (its block) is NaN, the others'
    norms are finite; an all-zero row with eps 0 is 0 / 0."""
    x = torch.randn(6, 64, generator=torch.Generator().manual_seed(2))
    x[0] *= 2.0 ** 100
    x[1, 5], x[2, 40], x[3] = float("inf"), float("nan"), 0.0
    x = x.bfloat16().to(cuda)
    zero, one = torch.zeros(6, 64, dtype=torch.bfloat16, device=cuda), torch.ones(64, device=cuda).bfloat16()
    *got, hidden = tm_ops.rms_norm_modulate_fp4_quant(x, one, 0.0, zero, zero, block_format=fmt,
                                                      return_hidden=True)
    nan = torch.isnan(hidden.cpu())
    assert nan[1, 5] and nan[2].all() and nan[3].all() and not nan[[0, 4, 5]].any()
    assert (hidden[1].cpu()[~nan[1]] == 0).all() and nan[1].sum() == 1
    _check_quant(got, hidden.cpu(), fmt)
    *_, hidden = tm_ops.rms_norm_modulate_fp4_quant(x, one, 1e-6, zero, zero, block_format=fmt,
                                                    return_hidden=True)
    assert (hidden[3] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("power", [-110, 110])
def test_given_scale_at_the_ends_of_its_range(tm_ops, cuda, dtype, power):
    given = 2.0 ** power
    x = torch.cat((_borders(dtype).double() * given, _borders(dtype).double() * given * 2.0 ** -9,
                   _borders(dtype).double() * 2.0 ** (power // 2))).to(dtype)
    got = tm_ops.scaled_fp4_quant(x.to(cuda), torch.tensor([given], device=cuda))
    _check_quant(got, x, "nvfp4", given)


@pytest.mark.parametrize("given", [0.0, -0.0, -1.0, float("nan"), float("inf"), 2.0 ** -111, 2.0 ** 111])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_given_scale_out_of_range_is_nan(tm_ops, cuda, dtype, given):
    """Every block scale is NaN and every code 0, in all-zero blocks too; the padding
    stays 0."""
    scale = torch.tensor([given], device=cuda)
    big = torch.randn(131, 33024, generator=torch.Generator().manual_seed(1)).to(dtype).to(cuda)
    big[3] = 0.0
    for x in (big[:, :96], big[:, 1:97], big[:2]):  # both kernels
        q, blocks, _ = tm_ops.scaled_fp4_quant(x, scale)
        rows, cols = x.shape
        want = np.zeros(blocks.numel(), dtype=np.uint8)
        want[f4.tile_offsets(rows, cols // 16)] = 0x7F
        np.testing.assert_array_equal(blocks.view(torch.uint8).cpu().numpy().reshape(-1), want)
        assert not q.any()
        assert torch.isnan(tm_ops.dequantize_fp4(q, blocks, scale)).all()


def test_allocating_operators_return_fresh_tensors(tm_ops, cuda):
    """The operators' outputs share no storage with an input, as their schemas say, a
    given scale among them; the Python call hands the given scale back itself."""
    raw = torch.ops.taomate_w8a8
    x = torch.randn(6, 64, device=cuda).bfloat16()
    scale = torch.tensor([0.01], device=cuda)
    w = tm_ops.scaled_fp4_quant(torch.randn(8, 64, device=cuda))
    q, b, s = tm_ops.scaled_fp4_quant(x)
    one = torch.ones(64, device=cuda).bfloat16()

    def check(op, args):
        outs = op.default(*args)
        storages = lambda ts: [t.untyped_storage().data_ptr() for t in ts  # noqa: E731
                               if isinstance(t, torch.Tensor)]
        outs = storages(outs if isinstance(outs, tuple) else (outs,))
        assert len(set(outs)) == len(outs) and not set(outs) & set(storages(args))

    check(raw.scaled_fp4_quant_new, (x, None, False))
    check(raw.scaled_fp4_quant_new, (x, None, True))
    check(raw.scaled_fp4_quant_new, (x, scale, False))
    assert raw.scaled_fp4_quant_new(x, scale, False)[2] is None
    # torch's own check of the schema (it takes no 8-bit floating-point inputs)
    torch.library.opcheck(raw.scaled_fp4_quant_new.default, (x, scale, False),
                          test_utils="test_schema")
    check(raw.dequantize_fp4_new, (q, b, s, torch.bfloat16))
    check(raw.scaled_mm_fp4_new, (q, w[0].t(), b, w[1], s, w[2], torch.bfloat16, None, 0))
    check(raw.modulate_fp4_quant_new, (x, x, x, None, False, True))
    check(raw.rms_norm_modulate_fp4_quant_new, (x, one, 1e-6, x, x, None, False, True))
    check(raw.residual_gate_rms_norm_modulate_fp4_quant_new,
          (x, x, x, one, 1e-6, x, x, None, False, True))
    got = tm_ops.scaled_fp4_quant(x, scale)
    assert got[2] is scale
    y = tm_ops.scaled_mm_fp4(got[0], w[0].t(), got[1], w[1], got[2], w[2])
    _check_mm(y, *got, *w, None, "nvfp4")


@pytest.mark.parametrize("tile,splits", [(0, 1), (32, 2), (128, 1), (1256, 1)])
def test_mm_leading_dimensions_under_every_tile(tm_ops, cuda, tile, splits):
    """[..., K / 2] codes give [..., N] whatever the kernel; `out` is returned as it is."""
    x = orc.activation(24, 512, 1, outlier_channels=None).bfloat16().to(cuda).view(2, 3, 4, 512)
    q, b, s = tm_ops.scaled_fp4_quant(x)
    w = tm_ops.scaled_fp4_quant(orc.weight(128, 512, seed=2).to(cuda))
    for swiglu, n in ((False, 128), (True, 64)):
        y = tm_ops.scaled_mm_fp4(q, w[0].t(), b, w[1], s, w[2], swiglu=swiglu, tile=tile,
                                 splits=splits)
        assert y.shape == (2, 3, 4, n)
        _check_mm(y.view(24, n), q.view(24, -1), b, s, *w, None, "nvfp4", "swiglu" if swiglu else "none")
        out = torch.empty(24, n, dtype=torch.bfloat16, device=cuda)
        assert tm_ops.scaled_mm_fp4(q, w[0].t(), b, w[1], s, w[2], swiglu=swiglu, out=out, tile=tile,
                                    splits=splits) is out
        assert torch.equal(out, y.view(24, n))
    empty = tm_ops.scaled_fp4_quant(x[:0])
    assert tm_ops.scaled_mm_fp4(empty[0], w[0].t(), empty[1], w[1], empty[2], w[2], tile=tile,
                                splits=splits).shape == (0, 3, 4, 128)


def _device_values(q, b, s, fmt):
    """_values for large tensors: the same by torch operations on the device."""
    rows, blocks = q.shape[0], q.shape[1] * 2 // f4.BLOCK[fmt]
    code = torch.stack((q & 15, q >> 4), -1).view(rows, blocks, -1).long()
    value = torch.tensor(np.concatenate((f4.E2M1, -f4.E2M1)), device=q.device)[code]
    at = torch.from_numpy(f4.tile_offsets(rows, blocks)).to(q.device)
    v = (value * b.float().double().view(-1)[at].unsqueeze(-1)).view(rows, -1)
    return (v if s is None else v * s.double().view(-1, 1)).cpu().numpy()


def _large_mm(tm_ops, cuda, monkeypatch, m, n, k, fmt, act, **forced):
    monkeypatch.setitem(globals(), "_values", _device_values)
    g = torch.Generator(device=cuda).manual_seed(m + n + k)
    rnd = lambda *shape: torch.randn(shape, generator=g, device=cuda)  # noqa: E731
    a = tm_ops.scaled_fp4_quant(rnd(m, k).bfloat16(), block_format=fmt)
    w = tm_ops.scaled_fp4_quant((rnd(n, k) * 0.03).bfloat16(), block_format=fmt)
    bias = (rnd(n) * 0.3).bfloat16()
    out = tm_ops.scaled_mm_fp4(a[0], w[0].t(), a[1], w[1], a[2], w[2], bias=bias,
                               gelu_tanh=act == "gelu", swiglu=act == "swiglu", **forced)
    _check_mm(out, *a, *w, bias, fmt, act)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("act", ["none", "gelu", "swiglu"])
@pytest.mark.parametrize("m,n,k", [
    (1, 20032, 2336), (33, 20032, 288), (128, 24000, 1056), (5, 40000, 544), (64, 19008, 96),
    (256, 9472, 608), (256, 9536, 608),   # 148 tiles of 128 x 128, and 150
    (129, 18944, 416), (1000, 2368, 800), (1000, 2432, 800),
])
def test_mm_more_tiles_than_sms(tm_ops, cuda, monkeypatch, m, n, k, act, fmt):
    """The chosen kernel where the small one has more tiles than the GPU has SMs (two
    blocks an SM, shorter rings), and on both sides of the change to the pair kernel."""
    _large_mm(tm_ops, cuda, monkeypatch, m, n, k, fmt, act)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tile,splits,m,n,k", [
    (32, 8, 20, 4160, 2336), (32, 2, 32, 12800, 800), (64, 4, 64, 8256, 1376), (128, 2, 300, 4160, 800),
    (128, 8, 300, 1344, 2336), (128, 4, 128, 6400, 1056),
])
def test_mm_slices_of_more_tiles_than_sms(tm_ops, cuda, monkeypatch, tile, splits, m, n, k, fmt):
    """Clusters of K slices in several waves, where two stages may exceed half an SM."""
    for act in ("none", "swiglu"):
        _large_mm(tm_ops, cuda, monkeypatch, m, n, k, fmt, act, tile=tile, splits=splits)
