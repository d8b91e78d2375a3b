"""Microscaled 4-bit floating point on the GPU against 64-bit numpy.

Tolerances.  Quantisation and dequantisation are exact up to the output's one rounding.  Products: n fp32 additions, each off by
at most 2^-23 of what has been summed (the tensor cores cut off instead of rounding), so n * 2^-23 * sum |x w|; then the result's
rounding, half a step: finfo.eps / 2 relative to the value (and half its smallest subnormal).
"""
import numpy as np
import pytest
import torch

import mx4_oracle as O
from glq_b200 import ops

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FORMATS = ["mxfp4", "nvfp4"]


def host(t):
    return t.detach().double().cpu().numpy()


def to_cuda(a, dtype=torch.float32):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda").to(dtype)


def check_quantized(x, fmt, t=None):
    """quantise x on the GPU and compare codes, scales and the tensor's scale with the oracle, bit for bit."""
    given = None if t is None else torch.tensor([t], dtype=torch.float32, device="cuda")
    q = ops.mx4_quantize(x, fmt, given)
    v = host(x).reshape(-1, x.shape[-1])
    if fmt == "nvfp4":
        ts = np.float32(O.tensor_scale(v)) if t is None else np.float32(t)
        assert q.tensor_scale.item() == ts
    else:
        ts = None
    code, byte = O.quantize(v, fmt, ts)
    got = O.unpack_nibbles(q.codes.cpu().numpy().reshape(len(v), -1), x.shape[-1])
    scales = q.scales.cpu().numpy().reshape(len(v), -1)
    assert np.array_equal(scales, byte)
    # (zeros may carry either sign)
    assert np.array_equal(np.where(got & 7, got, 0), np.where(code & 7, code, 0))
    if x.shape[-1] % 2:
        assert not (q.codes.cpu().numpy().reshape(len(v), -1)[:, -1] & 0xF0).any()
    return q


# ---- quantisation ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (2, 8), (5, 15), (1, 16), (4, 17), (3, 32), (2, 33), (7, 100), (64, 256), (13, 1000), (1, 2048), (300, 4100)])
def test_quantize_matches_definition(fmt, dtype, rows, cols):
    g = np.random.default_rng(rows * 10007 + cols)
    x = to_cuda(g.standard_normal((rows, cols)) * np.exp(g.standard_normal((rows, 1)) * 3), DT[dtype])
    q = check_quantized(x, fmt)
    assert q.codes.shape == (rows, (cols + 1) // 2) and q.cols == cols


@pytest.mark.parametrize("t", [1.0, 0.37, 2.0 ** -20, 1e-31, 3e-38, 1e30, 5e34])
def test_nvfp4_given_scale_and_ties(t):
    """Values on the borders of codes and of block scales: multiples of an eighth of the scale."""
    g = np.random.default_rng(5)
    x = (g.integers(-64, 65, (64, 160)) * 0.125) * np.float64(t)
    x[:, ::16] = np.float64(t) * 6 * O.E4M3[g.integers(40, 90, (64, 10))] * g.choice([1.0, 1.0625, 1.03125, 0.96875], (64, 10))
    check_quantized(to_cuda(x), "nvfp4", t)


def test_nvfp4_every_block_scale_border():
    """A block whose largest value lies on the middle between two e4m3 scales, and one fp32 step to either side."""
    middle = (O.E4M3[1:] + O.E4M3[:-1]) / 2
    for t in (1.0, 0.7):
        top = (6.0 * middle * np.float64(np.float32(t))).astype(np.float32)
        x = np.zeros((3 * len(top), 16), np.float32)
        x[0::3, 3], x[1::3, 3], x[2::3, 3] = top, np.nextafter(top, np.float32(0)), -np.nextafter(top, np.float32(np.inf))
        check_quantized(to_cuda(x), "nvfp4", t)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_extremes(fmt):
    x = np.zeros((10, 64), np.float32)
    x[0, 5] = np.inf
    x[1, 40] = np.nan
    x[2, :] = 3.4e38
    x[3, :] = np.float32(1e-45)
    x[4, ::3] = 1.1754944e-38
    x[5, 7] = -7.99
    x[6] = np.linspace(-6, 6, 64)
    x[7, 3], x[7, 4] = 1e30, 1e-30
    x[8, 0], x[8, 1] = -np.inf, np.nan
    for rows in (x, x[3:5], x[9:], x[5:7]):
        check_quantized(to_cuda(rows), fmt, None)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_strides_alignment_and_shapes(fmt):
    g = np.random.default_rng(1)
    base = to_cuda(g.standard_normal((40, 531)), torch.bfloat16)
    check_quantized(base[3:, 5:517], fmt)                       # rows that start on odd addresses
    check_quantized(base[:, :512], fmt)
    check_quantized(base[::2, 3:100], fmt)
    check_quantized(base.t(), fmt)                              # values apart
    check_quantized(base[0].expand(7, 531), fmt)                # the same row again
    check_quantized(base[:, :520].reshape(5, 8, 520), fmt)
    check_quantized(base[0], fmt)
    for shape in ((0, 64), (3, 0), (0,), (2, 0, 5)):
        q = ops.mx4_quantize(torch.zeros(shape, device="cuda"), fmt)
        assert q.codes.shape[:-1] == shape[:-1] and q.codes.numel() == 0
        assert ops.mx4_dequantize(q).shape == shape


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", [(1, 1), (3, 33), (8, 64), (5, 1001), (3, 4, 80)])
def test_dequantize_every_byte(fmt, dtype, shape):
    g = np.random.default_rng(shape[-1])
    cols, lead = shape[-1], shape[:-1]
    code = g.integers(0, 16, shape, dtype=np.uint8)
    byte = g.integers(0, 256 if fmt == "mxfp4" else 128, lead + (-(-cols // O.BLOCK[fmt]),), dtype=np.uint8)
    per = lead[0] if len(lead) == 2 else 1
    t = np.float32(g.uniform(0.1, 3, per)) if fmt == "nvfp4" else None
    q = ops.Mx4Tensor(to_cuda(O.pack_nibbles(code), torch.uint8), to_cuda(byte, torch.uint8), fmt, cols, to_cuda(t) if t is not None else None)
    got = ops.mx4_dequantize(q, DT[dtype])
    want = O.values(code, byte, fmt)
    if t is not None:
        want = (want.astype(np.float32) * t.reshape((per,) + (1,) * (want.ndim - 1))) if per > 1 else want.astype(np.float32) * t[0]
    with np.errstate(over="ignore"):
        want = torch.from_numpy(want.astype(np.float32)).to(DT[dtype])
    assert torch.equal(torch.nan_to_num(got.cpu(), nan=7.5), torch.nan_to_num(want, nan=7.5))


# ---- products --------------------------------------------------------------------------------------------------
def make_weight(g, shape, fmt, spread=1.0):
    """(packed weight, values in 64 bits (E, m, n) or (m, n))."""
    n = shape[-1]
    w = g.standard_normal(shape) * np.exp(g.standard_normal(shape[:-1] + (1,)) * spread) / np.sqrt(n)
    flat = w.reshape(-1, n)
    if fmt == "nvfp4":
        groups = shape[0] if len(shape) == 3 else 1
        t = np.array([O.tensor_scale(p) for p in flat.reshape(groups, -1, n)], np.float32)
        parts = [O.quantize(p, fmt, ti) for p, ti in zip(flat.reshape(groups, -1, n), t)]
        code, byte = np.concatenate([p[0] for p in parts]), np.concatenate([p[1] for p in parts])
        vals = np.concatenate([O.values(*p, fmt, ti) for p, ti in zip(parts, t)])
    else:
        t = None
        code, byte = O.quantize(flat, fmt)
        vals = O.values(code, byte, fmt)
    lead = shape[:-1]
    q = ops.Mx4Tensor(to_cuda(O.pack_nibbles(code).reshape(lead + (-1,)), torch.uint8), to_cuda(byte.reshape(lead + (-1,)), torch.uint8), fmt, n,
                      to_cuda(t) if t is not None else None)
    return ops.mx4_pack(q), vals.reshape(shape)


def quantized_values(x, fmt, t=None):
    ts = None if fmt == "mxfp4" else np.float32(O.tensor_scale(x) if t is None else t)
    return O.values(*O.quantize(x, fmt, ts), fmt, ts)


def tolerance(x, w, want, dtype):
    f = torch.finfo(dtype)
    return x.shape[-1] * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T) + f.eps / 2 * np.abs(want) + f.smallest_normal * f.eps / 2


def check_product(got, x, w, dtype, add=None):
    want = x @ w.T
    tol = tolerance(x, w, want if add is None else np.abs(want) + np.abs(add), dtype)
    if add is not None:
        want = want + add
    err = np.abs(host(got) - want)
    assert np.all(err <= tol), f"off by {np.nanmax(err / tol):.3g} tolerances at {np.unravel_index(np.argmax(err / tol), err.shape)}"


SIZES = [(1, 1, 1), (1, 128, 256), (1, 64, 64), (2, 130, 96), (1, 200, 1024), (3, 17, 33), (5, 300, 520), (8, 128, 2048), (9, 256, 256), (16, 384, 640),
         (17, 129, 257), (31, 128, 512), (33, 500, 1000), (64, 256, 768), (65, 128, 320), (100, 640, 512), (129, 130, 300), (192, 128, 256),
         (193, 257, 264), (300, 384, 1536), (513, 200, 144),
         (17, 256, 4400), (24, 130, 5000), (32, 2048, 1024), (32, 4300, 2100), (26, 136, 72)]


@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("tokens,m,n", SIZES)
def test_linear(fmt, dtype, quantize, tokens, m, n):
    g = np.random.default_rng(tokens * 1000003 + m * 1009 + n)
    weight, w = make_weight(g, (m, n), fmt)
    x = to_cuda(g.standard_normal((tokens, n)), DT[dtype])
    y = ops.mx4_linear(x, weight, quantize_input=quantize)
    assert y.shape == (tokens, m) and y.dtype == DT[dtype]
    xv = host(x)
    check_product(y, quantized_values(xv, fmt) if quantize else xv, w, DT[dtype])
    assert torch.equal(y, ops.mx4_linear(x, weight, quantize_input=quantize))      # no result depends on timing


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("tokens", [1, 20, 150])
@pytest.mark.parametrize("out", ["bf16", "fp16", "fp32"])
def test_linear_output_types_and_residual(fmt, quantize, tokens, out):
    g = np.random.default_rng(tokens)
    weight, w = make_weight(g, (272, 416), fmt)
    x = to_cuda(g.standard_normal((2, tokens, 416)), torch.bfloat16)
    xv = host(x).reshape(-1, 416)
    xq = quantized_values(xv, fmt) if quantize else xv
    y = ops.mx4_linear(x, weight, quantize_input=quantize, out_dtype=DT[out])
    assert y.shape == (2, tokens, 272) and y.dtype == DT[out]
    check_product(y.reshape(-1, 272), xq, w, DT[out])
    add = to_cuda(g.standard_normal((2, tokens, 272)), DT[out])
    before = host(add).reshape(-1, 272)
    r = ops.mx4_linear(x, weight, quantize_input=quantize, accumulate_into=add)
    assert r is add
    check_product(add.reshape(-1, 272), xq, w, DT[out], add=before)


@pytest.mark.parametrize("tokens", [2, 40, 200])
@pytest.mark.parametrize("quantize", [False, True])
def test_linear_strided_and_unaligned_rows(tokens, quantize):
    g = np.random.default_rng(tokens)
    weight, w = make_weight(g, (160, 328), "mxfp4")
    base = to_cuda(g.standard_normal((tokens, 700)), torch.bfloat16)
    for x in (base[:, :328], base[:, 8:336], base[:, 3:331], base[:, 1:657:2], base.t()[:328].t(), base[:1, :328].expand(tokens, 328)):
        xv = host(x)
        check_product(ops.mx4_linear(x, weight, quantize_input=quantize), quantized_values(xv, "mxfp4") if quantize else xv, w, torch.bfloat16)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("tokens", [3, 140])
def test_quantized_input_with_given_scale(dtype, tokens):
    g = np.random.default_rng(tokens)
    weight, w = make_weight(g, (144, 272), "nvfp4")
    x = to_cuda(g.standard_normal((tokens, 272)), DT[dtype])
    t = torch.tensor([0.0021], device="cuda")
    y = ops.mx4_linear(x, weight, quantize_input=True, input_scale=t)
    check_product(y, quantized_values(host(x), "nvfp4", t.item()), w, DT[dtype])


@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("tokens", [1, 24, 160])
def test_mxfp4_scales_over_the_whole_range(quantize, tokens):
    """Rows whose blocks have any exponent: 2^20 within a row, rows from 2^-127 to 2^100, a row of zeros, blocks that are NaN."""
    g = np.random.default_rng(3)
    m, n = 136, 512
    code = g.integers(0, 16, (m, n), dtype=np.uint8)
    base = np.linspace(0, 220, m).astype(int)[:, None]
    byte = np.clip(base + g.integers(0, 21, (m, n // 32)), 0, 254).astype(np.uint8)
    code[7] = 0
    byte[9, 3] = byte[m - 1, 15] = 255
    weight = ops.mx4_pack(ops.Mx4Tensor(to_cuda(O.pack_nibbles(code), torch.uint8), to_cuda(byte, torch.uint8), "mxfp4", n))
    w = O.values(code, byte, "mxfp4")
    for dtype in (torch.bfloat16, torch.float16):
        x = to_cuda(g.standard_normal((tokens, n)) * 2.0 ** -3, dtype)
        xv = quantized_values(host(x), "mxfp4") if quantize else host(x)
        y = ops.mx4_linear(x, weight, quantize_input=quantize, out_dtype=torch.float32)
        got = host(y)
        nan = np.zeros(m, bool)
        nan[[9, m - 1]] = True
        assert np.isnan(got[:, nan]).all() and np.isfinite(got[:, ~nan]).all()
        # (sums of the smallest rows are subnormal in fp32: each addition may lose half of 2^-149; half of them are cut off)
        wz = np.where(nan[:, None], 0.0, w)
        want = xv @ wz.T
        tol = tolerance(xv, wz, want, torch.float32) + n * 2.0 ** -149
        # products below 2^-126 may be taken as zero by the matrix instructions
        tol = tol + n * 2.0 ** -126 * (np.abs(w).max(1, initial=0.0, where=~np.isnan(w)) < 2.0 ** -100)
        assert np.all(np.abs(got - want)[:, ~nan] <= tol[:, ~nan])


# ---- grouped by expert ------------------------------------------------------------------------------------------
def counts_to_offsets(counts, first=0, dtype=torch.int32):
    return torch.tensor(np.concatenate([[first], first + np.cumsum(counts)]), dtype=dtype, device="cuda")


COUNTS = {
    "one_each": [1] * 7,
    "some_empty": [0, 3, 0, 0, 17, 1, 0],
    "one_takes_all": [0, 0, 70, 0],
    "none": [0, 0, 0],
    "ragged": [5, 130, 16, 64, 1, 33, 193, 2],
    "one_expert": [50],
    "many": [1, 0, 2, 0, 3] * 30,
    "large": [300, 0, 129, 260],
}


@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("name", list(COUNTS))
def test_grouped(fmt, quantize, name):
    counts = COUNTS[name]
    g = np.random.default_rng(len(counts))
    m, n = (200, 352) if len(counts) < 20 else (130, 96)
    dtype = torch.bfloat16 if fmt == "mxfp4" else torch.float16
    weight, w = make_weight(g, (len(counts), m, n), fmt)
    first, behind = 3, 5
    rows = sum(counts) + first + behind
    xh = g.standard_normal((rows, n))
    xh[:first] = np.nan                                          # rows of no expert are not read into anything
    xh[rows - behind:] = 1e4
    x = to_cuda(xh, dtype)
    off = counts_to_offsets(counts, first, torch.int64 if len(counts) % 2 else torch.int32)
    y = ops.mx4_grouped_linear(x, weight, off, quantize_input=quantize)
    at = off.tolist()
    assert not y[:first].any() and not y[at[-1]:].any()
    xv = host(x)[first:at[-1]]
    if quantize and len(xv):
        xv = quantized_values(xv, fmt)
    for e in range(len(counts)):
        if counts[e]:
            check_product(y[at[e]:at[e + 1]], xv[at[e] - first:at[e + 1] - first], w[e], dtype)
    # a given result keeps the rows of no expert, also with rows that lie apart
    out = torch.full((rows, m + 9), 7.0, dtype=dtype, device="cuda")
    r = ops.mx4_grouped_linear(x, weight, off, quantize_input=quantize, out=out[:, 4:4 + m])
    assert r.data_ptr() == out[:, 4:].data_ptr()
    assert torch.equal(out[first:at[-1], 4:4 + m], y[first:at[-1]])
    out[first:at[-1], 4:4 + m] = 7.0
    assert (out == 7.0).all()


@pytest.mark.parametrize("quantize", [False, True])
def test_grouped_offsets_that_make_no_sense_stay_in_bounds(quantize):
    g = np.random.default_rng(2)
    weight, w = make_weight(g, (4, 144, 160), "mxfp4")
    x = to_cuda(g.standard_normal((60, 160)), torch.bfloat16)
    xv = quantized_values(host(x), "mxfp4") if quantize else host(x)
    for off in ([-5, 10, 10, 30, 1000], [0, 40, 20, 60, 60], [100, 200, 300, 400, 500], [-9, -8, -7, -6, -5], [0, 2 ** 40, 2 ** 41, 5, 60]):
        y = ops.mx4_grouped_linear(x, weight, torch.tensor(off, dtype=torch.int64, device="cuda"), quantize_input=quantize)
        seen = np.zeros(60, bool)
        for e in range(4):
            b, f = (min(max(v, 0), 60) for v in off[e:e + 2])
            alone = [k for k in range(b, f) if sum(min(max(off[i], 0), 60) <= k < min(max(off[i + 1], 0), 60) for i in range(4)) == 1]
            if alone:
                check_product(y[alone], xv[alone], w[e], torch.bfloat16)
            seen[b:max(b, f)] = True
        assert not host(y)[~seen].any()


def test_grouped_matches_linear_per_expert():
    g = np.random.default_rng(8)
    counts = [40, 0, 25, 90]
    weight, w = make_weight(g, (4, 256, 512), "nvfp4")
    x = to_cuda(g.standard_normal((sum(counts), 512)), torch.bfloat16)
    off = counts_to_offsets(counts)
    y = ops.mx4_grouped_linear(x, weight, off, out_dtype=torch.float32)
    at = off.tolist()
    for e in range(4):
        if counts[e]:
            check_product(y[at[e]:at[e + 1]], host(x)[at[e]:at[e + 1]], w[e], torch.float32)


# ---- streams, graphs, together ------------------------------------------------------------------------------------
@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("tokens", [1, 30, 140])
def test_captured_and_replayed_with_new_inputs(quantize, tokens):
    g = np.random.default_rng(4)
    weight, w = make_weight(g, (256, 384), "nvfp4")
    experts, we = make_weight(g, (3, 256, 384), "nvfp4")
    x = to_cuda(g.standard_normal((tokens, 384)), torch.bfloat16)
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):                                       # two graphs of the same calls, replayed at once below
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                y = ops.mx4_linear(x, weight, quantize_input=quantize)
                z = ops.mx4_grouped_linear(x, experts, off, quantize_input=quantize)
                v = ops.mx4_dequantize(ops.mx4_quantize(x, "nvfp4"), torch.float32)
            graphs.append((graph, y, z, v))
    torch.cuda.current_stream().wait_stream(side)
    for k in range(3):
        x.copy_(to_cuda(g.standard_normal((tokens, 384)) * (k + 1), torch.bfloat16))
        cut = sorted(g.integers(0, tokens + 1, 2).tolist())
        off.copy_(torch.tensor([0] + cut + [tokens], dtype=torch.int32))
        torch.cuda.synchronize()
        other = torch.cuda.Stream()
        graphs[0][0].replay()
        with torch.cuda.stream(other):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        xv = host(x)
        xq = quantized_values(xv, "nvfp4")
        for _, y, z, v in graphs:
            check_product(y, xq if quantize else xv, w, torch.bfloat16)
            at = [0] + cut + [tokens]
            for e in range(3):
                if at[e] < at[e + 1]:
                    check_product(z[at[e]:at[e + 1]], (xq if quantize else xv)[at[e]:at[e + 1]], we[e], torch.bfloat16)
            assert np.allclose(host(v), xq, rtol=2.0 ** -23, atol=0)
    ops.check_device_status()


def test_calls_on_several_streams_at_once():
    g = np.random.default_rng(6)
    weight, w = make_weight(g, (512, 1024), "mxfp4")
    xs = [to_cuda(g.standard_normal((t, 1024)), torch.bfloat16) for t in (1, 7, 48, 130, 300)]
    torch.cuda.synchronize()
    for quantize in (False, True):
        alone = [ops.mx4_linear(x, weight, quantize_input=quantize) for x in xs]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in xs]
        got = [[] for _ in xs]
        for _ in range(10):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i].append(ops.mx4_linear(xs[i], weight, quantize_input=quantize))
        torch.cuda.synchronize()
        for i in range(len(xs)):
            assert all(torch.equal(y, alone[i]) for y in got[i])


def test_calls_of_every_form_behind_one_another():
    """Chained launches of all forms in changing order, on one stream and on three: the bits of each call alone."""
    g = np.random.default_rng(21)
    torch.manual_seed(21)
    sizes = ((512, 1024), (2048, 2048), (1100, 648))
    weights = {(f, s): ops.mx4_pack(ops.mx4_quantize(torch.randn(s, device="cuda"), f)) for f in FORMATS for s in sizes + ((16, 640, 512),)}

    def job(fmt, quantize, tokens, dtype):
        if g.random() < 0.3:
            counts = g.integers(0, max(1, tokens // 8) + 1, 16)
            off, x = counts_to_offsets(counts), torch.randn(int(counts.sum()) + 2, 512, device="cuda", dtype=dtype)
            return lambda: ops.mx4_grouped_linear(x, weights[fmt, (16, 640, 512)], off, quantize_input=quantize)
        m, n = sizes[g.integers(len(sizes))]
        x = torch.randn(tokens, n, device="cuda", dtype=dtype)
        return lambda: ops.mx4_linear(x, weights[fmt, (m, n)], quantize_input=quantize)

    jobs = [job(f, q, t, d) for f in FORMATS for q in (False, True) for t in (1, 16, 20, 33, 150, 2100) for d in (torch.bfloat16, torch.float16)]
    alone = []
    for j in jobs:
        alone.append(j())
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for turn in range(10):
        got = {int(i): jobs[i]() for i in g.permutation(len(jobs))}
        torch.cuda.synchronize()
        assert all(torch.equal(got[i], alone[i]) for i in got)
        for i in g.permutation(len(jobs)):
            with torch.cuda.stream(streams[i % 3]):
                got[int(i)] = jobs[i]()
        torch.cuda.synchronize()
        assert all(torch.equal(got[i], alone[i]) for i in got)
    ops.check_device_status()


@pytest.mark.parametrize("fmt", FORMATS)
def test_experts_layer_of_a_decoder(fmt):
    """The operators as they are used together: a dense block with residual, then routed experts over sorted rows."""
    g = np.random.default_rng(9)
    hidden, inter, experts, tokens, top = 256, 192, 6, 50, 2
    up, wu = make_weight(g, (2 * inter, hidden), fmt, spread=0.2)
    down, wd = make_weight(g, (hidden, inter), fmt, spread=0.2)
    w13, v13 = make_weight(g, (experts, 2 * inter, hidden), fmt, spread=0.2)
    w2, v2 = make_weight(g, (experts, hidden, inter), fmt, spread=0.2)
    x = to_cuda(g.standard_normal((tokens, hidden)), torch.bfloat16)

    def act(h):
        return torch.nn.functional.silu(h[:, :inter]) * h[:, inter:]

    res = x.clone()
    h = ops.mx4_linear(x, up, out_dtype=torch.float32)
    check_product(h, host(x), wu, torch.float32)
    a = act(h).to(torch.bfloat16)
    before = host(res)
    ops.mx4_linear(a, down, accumulate_into=res)
    check_product(res, host(a), wd, torch.bfloat16, add=before)
    ids = torch.from_numpy(np.stack([g.permutation(experts)[:top] for _ in range(tokens)])).cuda()
    weights = torch.rand(tokens, top, device="cuda")
    order = torch.argsort(ids.flatten(), stable=True)
    token = order // top
    off = torch.cat((ids.new_zeros(1), torch.bincount(ids.flatten(), minlength=experts).cumsum(0))).to(torch.int32)
    rows = res[token]
    h = ops.mx4_grouped_linear(rows, w13, off, out_dtype=torch.float32)
    a = act(h).to(torch.bfloat16)
    y = ops.mx4_grouped_linear(a, w2, off, out_dtype=torch.float32)
    out = torch.zeros(tokens, hidden, device="cuda").index_add_(0, token, y * weights.flatten()[order, None])
    want = np.zeros((tokens, hidden))
    at = off.tolist()
    for e in range(experts):
        r = slice(at[e], at[e + 1])
        check_product(h[r], host(rows)[r], v13[e], torch.float32)
        part = host(a)[r] @ v2[e].T
        check_product(y[r], host(a)[r], v2[e], torch.float32)
        np.add.at(want, token[r].cpu().numpy(), part * host(weights.flatten()[order][r])[:, None])
    assert np.allclose(host(out), want, rtol=1e-4, atol=1e-4 * np.abs(want).max())
    ops.check_device_status()


# ---- forms that only larger calls take ---------------------------------------------------------------------------
@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("tokens,m,n", [(1500, 1024, 384), (1921, 1100, 640), (2048, 1153, 96), (3000, 900, 264)])
def test_linear_of_many_tokens(fmt, dtype, quantize, tokens, m, n):
    """Two CTAs to a tile of 256 weight rows, also an odd number of them, with values that end inside a step."""
    g = np.random.default_rng(tokens + m + n)
    weight, w = make_weight(g, (m, n), fmt)
    x = to_cuda(g.standard_normal((tokens, n)), DT[dtype])
    y = ops.mx4_linear(x, weight, quantize_input=quantize)
    xv = quantized_values(host(x), fmt) if quantize else host(x)
    check_product(y, xv, w, DT[dtype])
    assert torch.equal(y, ops.mx4_linear(x, weight, quantize_input=quantize))
    add = torch.zeros_like(y)
    ops.mx4_linear(x, weight, quantize_input=quantize, accumulate_into=add)
    assert torch.equal(add, y)


@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("experts,per,m,n", [(100, 20, 300, 160), (40, 90, 270, 96), (12, 300, 1100, 128), (1024, 1, 130, 64), (1024, 11, 16, 40)])
def test_grouped_many_experts(fmt, quantize, experts, per, m, n):
    """More tiles than CTAs, by one CTA each and by two, with counts from none to four times the average."""
    g = np.random.default_rng(experts)
    weight, w = make_weight(g, (experts, m, n), fmt)
    counts = g.multinomial(experts * per, g.dirichlet(np.full(experts, 1.5)))
    counts[[0, 5]] = 0
    x = to_cuda(g.standard_normal((int(counts.sum()), n)), torch.bfloat16)
    off = counts_to_offsets(counts)
    y = ops.mx4_grouped_linear(x, weight, off, quantize_input=quantize)
    xv = quantized_values(host(x), fmt) if quantize else host(x)
    at = off.tolist()
    for e in range(experts):
        if counts[e]:
            check_product(y[at[e]:at[e + 1]], xv[at[e]:at[e + 1]], w[e], torch.bfloat16)
    assert torch.equal(y, ops.mx4_grouped_linear(x, weight, off, quantize_input=quantize))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens", [1, 7, 16, 40, 250])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_activations_of_any_size(fmt, tokens, dtype):
    """Rows of x between 2^-100 and 2^100 (fp16: 2^-14 and 2^12), mixed magnitudes in a row, infinities and NaN, which stay in their rows."""
    g = np.random.default_rng(tokens)
    m, n = 200, 600
    weight, w = make_weight(g, (m, n), fmt, spread=0.1)
    span = np.linspace(-100, 100, tokens) if dtype == "bf16" else np.linspace(-14, 8, tokens)
    x = g.standard_normal((tokens, n)) * 2.0 ** span[:, None] * 2.0 ** g.integers(-12, 1, (tokens, n))
    bad = sorted({0, tokens // 2, tokens - 1}) if tokens > 1 else []
    for r, value in zip(bad, (np.inf, -np.inf, np.nan)):
        x[r, 300 + r % 200] = value
    if tokens > 6:
        x[3] = 0.0
    xd = to_cuda(x, DT[dtype])
    xv = host(xd)
    y = host(ops.mx4_linear(xd, weight, out_dtype=torch.float32))
    clean = np.setdiff1d(np.arange(tokens), bad)
    want = xv[clean] @ w.T
    # bf16 values may be multiplied as fp16 under a power of two per 256 of them: off by 2^-40 of the largest
    low = 2.0 ** -40 * n * np.abs(xv[clean]).max(1, keepdims=True, initial=0) * np.abs(w).max(1)
    assert np.all(np.abs(y[clean] - want) <= tolerance(xv[clean], w, want, torch.float32) + low)
    for r in bad:
        with np.errstate(invalid="ignore"):
            terms = xv[r] * w
            want_bad = terms.sum(1)
        assert np.array_equal(np.isnan(y[r]), np.isnan(want_bad)) and np.array_equal(np.isposinf(y[r]), np.isposinf(want_bad))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens,m", [(1, 200), (40, 200), (250, 200), (1700, 1100)])
def test_quantized_activations_with_infinities_and_nan(fmt, tokens, m):
    """A block that holds one becomes NaN, and with it its row of the result; the others are what they are without it."""
    g = np.random.default_rng(tokens)
    n = 328
    weight, w = make_weight(g, (m, n), fmt)
    x = g.standard_normal((tokens, n))
    bad = sorted({0, tokens // 3, tokens - 1})
    for r, value in zip(bad, (np.nan, np.inf, -np.inf)):
        x[r, (r * 7) % n] = value
    xd = to_cuda(x, torch.bfloat16)
    y = host(ops.mx4_linear(xd, weight, quantize_input=True, out_dtype=torch.float32))
    assert np.isnan(y[bad]).all()
    clean = np.setdiff1d(np.arange(tokens), bad)
    if len(clean):
        xv = quantized_values(host(xd), fmt)[clean]
        want = xv @ w.T
        assert np.all(np.abs(y[clean] - want) <= tolerance(xv, w, want, torch.float32))


@pytest.mark.parametrize("fmt", FORMATS)
def test_weights_with_nan_blocks_and_an_expert_of_zeros(fmt):
    """NaN blocks of weights stay in their rows, in every form; an expert whose weights are all zero gives zeros."""
    g = np.random.default_rng(2)
    experts, m, n = 3, 140, 288
    dense = g.standard_normal((experts, m, n))
    dense[1] = 0.0
    dense[0, 5, 40] = np.nan
    dense[2, 139, 287] = np.inf
    q = ops.mx4_quantize(to_cuda(dense), fmt)
    weight = ops.mx4_pack(q)
    nan = np.zeros((experts, m), bool)
    nan[0, 5] = nan[2, 139] = True
    w = host(ops.mx4_dequantize(q, torch.float32))
    assert np.array_equal(np.isnan(w).any(-1), nan)
    for per in (3, 50, 200):
        off = counts_to_offsets([per] * experts)
        x = to_cuda(g.standard_normal((experts * per, n)), torch.bfloat16)
        for quantize in (False, True):
            y = host(ops.mx4_grouped_linear(x, weight, off, quantize_input=quantize, out_dtype=torch.float32))
            xv = quantized_values(host(x), fmt) if quantize else host(x)
            for e in range(experts):
                r = slice(e * per, (e + 1) * per)
                assert np.isnan(y[r][:, nan[e]]).all()
                want = xv[r] @ w[e][~nan[e]].T
                assert np.all(np.abs(y[r][:, ~nan[e]] - want) <= tolerance(xv[r], w[e][~nan[e]], want, torch.float32))


def test_stored_rows_that_start_anywhere():
    """Codes and scales in views that begin on odd addresses."""
    g = np.random.default_rng(4)
    for fmt in FORMATS:
        q = ops.mx4_quantize(to_cuda(g.standard_normal((37, 203))), fmt)
        for shift in (1, 2, 5):
            codes, scales = (torch.zeros(t.numel() + shift, dtype=torch.uint8, device="cuda")[shift:].view(t.shape).copy_(t) for t in (q.codes, q.scales))
            moved = q._replace(codes=codes, scales=scales)
            assert torch.equal(ops.mx4_dequantize(moved), ops.mx4_dequantize(q))
            assert torch.equal(ops.mx4_pack(moved).image, ops.mx4_pack(q).image)


@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("tokens", [1, 60])
def test_weights_packed_right_in_front_of_the_product(quantize, tokens):
    """Weights written by the launch in front of a product are the ones it multiplies, eager and in a graph."""
    g = np.random.default_rng(6)
    m, n = 1024, 2048
    dense = [to_cuda(g.standard_normal((m, n)), torch.bfloat16) for _ in range(3)]
    x = to_cuda(g.standard_normal((tokens, n)), torch.bfloat16)
    want = []
    for d in dense:
        w = ops.mx4_pack(ops.mx4_quantize(d))
        torch.cuda.synchronize()
        want.append(ops.mx4_linear(x, w, quantize_input=quantize))
    images = [ops.mx4_pack(ops.mx4_quantize(d)).image for d in dense]
    assert not torch.equal(want[0], want[1])
    source = dense[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.mx4_linear(x, ops.mx4_pack(ops.mx4_quantize(source)), quantize_input=quantize)
    w = ops.mx4_pack(ops.mx4_quantize(dense[0]))
    for _ in range(5):
        for d, image, right in zip(dense, images, want):
            assert torch.equal(ops.mx4_linear(x, ops.mx4_pack(ops.mx4_quantize(d)), quantize_input=quantize), right)
            w.image.copy_(image)
            assert torch.equal(ops.mx4_linear(x, w, quantize_input=quantize), right)
            source.copy_(d)
            graph.replay()
            assert torch.equal(y, right)


def test_offsets_beyond_32_bits():
    """More than 2^31 values in x and in the result."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    g = np.random.default_rng(1)
    rows, cols = 135000, 16384
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    tail = to_cuda(g.standard_normal((70, cols)), torch.bfloat16)
    x[-70:] = tail
    for fmt in FORMATS:
        q, alone = ops.mx4_quantize(x, fmt), ops.mx4_quantize(tail, fmt)
        assert torch.equal(q.codes[-70:], alone.codes) and torch.equal(q.scales[-70:], alone.scales)
        assert torch.equal(ops.mx4_dequantize(q)[-70:], ops.mx4_dequantize(alone))
        assert not q.codes[:-70].any()
        del q
    weight, w = make_weight(g, (128, cols), "mxfp4")
    for quantize in (False, True):
        y = ops.mx4_linear(x, weight, quantize_input=quantize)
        check_product(y[-70:], quantized_values(host(tail), "mxfp4") if quantize else host(tail), w, torch.bfloat16)
        assert not y[:-70].any()
    del x, y
    torch.cuda.empty_cache()
    weight, w = make_weight(g, (cols, 64), "nvfp4")
    x = torch.zeros(rows, 64, dtype=torch.bfloat16, device="cuda")
    x[-70:] = tail[:, :64]
    for quantize in (False, True):
        y = ops.mx4_linear(x, weight, quantize_input=quantize)
        check_product(y[-70:], quantized_values(host(tail[:, :64]), "nvfp4") if quantize else host(tail[:, :64]), w, torch.bfloat16)
        assert not y[:-70].any()


def test_more_sixteens_than_31_bits():
    """Rows whose sixteens of values are counted in 64 bits."""
    rows, cols = 8330000, 4100
    if torch.cuda.mem_get_info()[0] < 110 << 30:
        pytest.skip("needs 110 GB")
    g = np.random.default_rng(1)
    tail = to_cuda(g.standard_normal((9, cols)), torch.bfloat16)
    for fmt in FORMATS:
        x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
        x[-9:] = tail
        q, alone = ops.mx4_quantize(x, fmt), ops.mx4_quantize(tail, fmt)
        del x
        assert torch.equal(q.codes[-9:], alone.codes) and torch.equal(q.scales[-9:], alone.scales)
        y = ops.mx4_dequantize(q)
        assert torch.equal(y[-9:], ops.mx4_dequantize(alone)) and not y[-10].any() and not y[0].any()
        del y, q
    torch.cuda.empty_cache()


@pytest.mark.parametrize("fmt", FORMATS)
def test_layer_of_4_bit_weights(fmt):
    import copy
    from glq_b200.linear import Mx4Linear
    g = np.random.default_rng(12)
    dense, bias = to_cuda(g.standard_normal((96, 160)) / 12), to_cuda(g.standard_normal(96))
    layer = Mx4Linear.from_weight(dense, bias, fmt)
    x = to_cuda(g.standard_normal((3, 5, 160)), torch.bfloat16)
    y = layer(x)
    assert y.shape == (3, 5, 96)
    direct = ops.mx4_linear(x, ops.mx4_pack(ops.mx4_quantize(dense, fmt)))
    assert torch.equal(y, direct + bias.to(torch.bfloat16))
    assert torch.equal(layer.dequantize(), ops.mx4_dequantize(ops.mx4_quantize(dense, fmt), torch.float32))
    assert layer.weight is layer.weight and not layer.codes.is_cpu
    # another layer loads it, after it has run with what it held before
    other = Mx4Linear(160, 96, bias=True, format=fmt).cuda()
    assert torch.equal(other(x), torch.zeros_like(y))
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), y)
    other.codes[:48].zero_()
    assert torch.equal(other(x)[..., :48], torch.zeros_like(y[..., :48]) + bias[:48].to(torch.bfloat16))
    twin = copy.deepcopy(layer)
    assert torch.equal(twin(x), y) and twin.weight is not layer.weight
    twin.quantize_input = True
    assert torch.equal(twin(x.float()), ops.mx4_linear(x.float(), layer.weight, quantize_input=True) + bias)
    twin.half()
    assert twin.bias.dtype == torch.float32 and torch.equal(layer(x), y)


# ---- refusals ----------------------------------------------------------------------------------------------------
def test_refusals():
    g = np.random.default_rng(0)
    weight, _ = make_weight(g, (64, 96), "mxfp4")
    nv, _ = make_weight(g, (64, 96), "nvfp4")
    experts, _ = make_weight(g, (2, 64, 96), "mxfp4")
    x = torch.zeros(4, 96, dtype=torch.bfloat16, device="cuda")
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    one = torch.ones(1, device="cuda")

    def refuse(match, call, kind=(ValueError, RuntimeError)):
        with pytest.raises(kind, match=match):
            call()

    refuse("inputs", lambda: ops.mx4_linear(x[:, :64], weight))
    refuse("fp32", lambda: ops.mx4_linear(x.float(), weight))
    refuse("not torch.int32", lambda: ops.mx4_linear(x.int(), weight))
    refuse("one per expert", lambda: ops.mx4_linear(x, experts))
    refuse("one matrix per expert", lambda: ops.mx4_grouped_linear(x, weight, off))
    refuse("3 int32 or int64", lambda: ops.mx4_grouped_linear(x, experts, off[:2]))
    refuse("3 int32 or int64", lambda: ops.mx4_grouped_linear(x, experts, off.float()))
    refuse("CUDA tensor", lambda: ops.mx4_grouped_linear(x, experts, off.cpu()))
    refuse("CUDA tensor", lambda: ops.mx4_linear(x.cpu(), weight))
    refuse("rows, n", lambda: ops.mx4_grouped_linear(x[None], experts, off))
    refuse("out must be", lambda: ops.mx4_grouped_linear(x, experts, off, out=torch.zeros(4, 63, device="cuda")))
    refuse("out overlaps", lambda: ops.mx4_grouped_linear(x, experts, off, out=x[:, :64]))
    refuse("input_scale", lambda: ops.mx4_linear(x, weight, quantize_input=True, input_scale=one))
    refuse("input_scale", lambda: ops.mx4_linear(x, nv, input_scale=one))
    refuse("1 fp32 value", lambda: ops.mx4_linear(x, nv, quantize_input=True, input_scale=one.double()))
    refuse("dense", lambda: ops.mx4_linear(x, weight, accumulate_into=torch.zeros(4, 70, device="cuda")[:, :64]))
    refuse("out_dtype", lambda: ops.mx4_linear(x, weight, accumulate_into=torch.zeros(4, 64, device="cuda"), out_dtype=torch.bfloat16))
    square, _ = make_weight(g, (96, 96), "mxfp4")
    refuse("overlaps x", lambda: ops.mx4_linear(x, square, accumulate_into=x))
    refuse("tensor_scale", lambda: ops.mx4_quantize(x, "mxfp4", one))
    refuse("not torch.float64", lambda: ops.mx4_quantize(x.double()))
    q = ops.mx4_quantize(x)
    refuse("are not mxfp4 rows", lambda: ops.mx4_pack(q._replace(cols=64)))
    refuse("needs its tensor_scale", lambda: ops.mx4_pack(ops.mx4_quantize(x, "nvfp4")._replace(tensor_scale=None)))
    refuse("tensor scales", lambda: ops.mx4_pack(ops.mx4_quantize(x, "nvfp4")._replace(tensor_scale=torch.ones(3, device="cuda"))))
    refuse("uint8", lambda: ops.mx4_dequantize(q._replace(codes=q.codes.int())))
    refuse("empty", lambda: ops.mx4_pack(ops.mx4_quantize(x[:0])))
    assert ops.mx4_linear(x[:0], weight).shape == (0, 64)
    assert ops.mx4_grouped_linear(x[:0], experts, off * 0).shape == (0, 64)
    with pytest.raises(AttributeError, match="cannot be set"):
        weight.image = weight.image.clone()
    scale = torch.tensor([0.5], device="cuda")
    own = ops.mx4_pack(ops.mx4_quantize(x, "nvfp4", scale))
    scale.fill_(2.0)
    assert own.tensor_scale.item() == 0.5


# ---- offsets out of order, and the scale of 4-bit activations ------------------------------------------------------
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
@pytest.mark.parametrize("off", [[0, 20, 60, 50], [5, 60, 10, 0], [0, 0, 40, -3], [70, 10, 20, 30], [0, 30, 45, 60], [9, 9, 9, 9]])
def test_scale_of_grouped_inputs_is_that_of_the_rows_multiplied(off, wide):
    """An offset below one before it counts as that one: rows behind the last offset as it is written are some expert's, and the
    largest values among them set the scale.  Rows of no expert do not."""
    g = np.random.default_rng(14)
    weight, w = make_weight(g, (3, 144, 160), "nvfp4")
    xh = g.standard_normal((64, 160))
    edge = np.maximum.accumulate(np.clip(off, 0, 64))
    xh[edge[-1]:] = 1e3                                           # of no expert
    xh[:edge[0]] = -1e3
    if edge[-1] > edge[0]:
        xh[edge[-1] - 1, 7] = 60.0
    x = to_cuda(xh, torch.bfloat16)
    y = ops.mx4_grouped_linear(x, weight, torch.tensor(off, dtype=wide, device="cuda"), quantize_input=True)
    assert not y[:edge[0]].any() and not y[edge[-1]:].any()
    if edge[-1] == edge[0]:
        return
    xv = quantized_values(host(x)[edge[0]:edge[-1]], "nvfp4")
    for e in range(3):
        if edge[e] < edge[e + 1]:
            check_product(y[edge[e]:edge[e + 1]], xv[edge[e] - edge[0]:edge[e + 1] - edge[0]], w[e], torch.bfloat16)


# ---- the layer on several streams ------------------------------------------------------------------------------------
DELAY = 40_000_000                  # clocks that a stream is kept busy: some 20 ms


def layers_and_input(fmt="mxfp4", seed=15):
    """Two layers of the same sizes and their results for x, each alone."""
    from glq_b200.linear import Mx4Linear
    g = np.random.default_rng(seed)
    layers = [Mx4Linear.from_weight(to_cuda(g.standard_normal((1024, 2048)) / 45), None, fmt) for _ in range(2)]
    x = to_cuda(g.standard_normal((20, 2048)), torch.bfloat16)
    want = [ops.mx4_linear(x, ops.mx4_pack(layer._rows())) for layer in layers]
    torch.cuda.synchronize()
    assert not torch.equal(*want)
    return layers, x, want


@pytest.mark.parametrize("fmt", FORMATS)
def test_layer_packed_on_one_stream_and_read_on_another(fmt):
    (layer, other), x, want = layers_and_input(fmt)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        torch.cuda._sleep(DELAY)
        ya = layer(x)
    with torch.cuda.stream(b):
        yb = layer(x)
    torch.cuda.synchronize()
    assert torch.equal(ya, want[0]) and torch.equal(yb, want[0])
    # b is late: what it reads must still be there after the layer has been packed again, and after it has gone
    for change in (lambda: layer.load_state_dict(other.state_dict()), lambda: layer.codes.copy_(other.codes), layer.half, layer.repack):
        layer.load_state_dict(layers_and_input(fmt)[0][0].state_dict())
        layer(x)
        with torch.cuda.stream(b):
            torch.cuda._sleep(DELAY)
            yb = layer(x)
        with torch.cuda.stream(a):
            change()
            ya = layer(x)
            junk = torch.full_like(layer.weight.image, 0x55)
        torch.cuda.synchronize()
        assert torch.equal(yb, want[0])
        assert torch.equal(ya, ops.mx4_linear(x, ops.mx4_pack(layer._rows())))
        del junk


def test_layer_that_goes_while_another_stream_reads_it():
    (layer, _), x, want = layers_and_input()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        size = layer.weight.image.numel()
    with torch.cuda.stream(b):
        torch.cuda._sleep(DELAY)
        y = layer(x)
    del layer
    with torch.cuda.stream(a):
        junk = [torch.full((size,), 0x55, dtype=torch.uint8, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    assert torch.equal(y, want[0])
    del junk


@pytest.mark.parametrize("fmt", FORMATS)
def test_captured_layer_whose_weights_change(fmt):
    """A graph goes on with the memory that it was captured with: the layer's weight of the day, packed by a forward or by `weight`."""
    (layer, other), x, want = layers_and_input(fmt)
    layer(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x)
    held, at = layer.weight, layer.weight.image.data_ptr()
    stored = {k: v.clone() for k, v in layer.state_dict().items()}
    for state, right in ((other.state_dict(), want[1]), (stored, want[0]), (other.state_dict(), want[1])):
        layer.load_state_dict(state)
        assert torch.equal(layer(x), right)
        assert layer.weight is held and held.image.data_ptr() == at
        junk = torch.full_like(held.image, 0x55)
        graph.replay()
        assert torch.equal(y, right)
        del junk
    with torch.inference_mode():
        layer.load_state_dict(stored)
        layer.repack()
        assert torch.equal(layer(x), want[0])
    graph.replay()
    assert layer.weight is held and torch.equal(y, want[0])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("experts", [None, 3])
def test_packing_into_a_packed_weight(fmt, experts):
    g = np.random.default_rng(17)
    shape = (150, 328) if experts is None else (experts, 150, 328)

    def stored():
        q = ops.mx4_quantize(to_cuda(g.standard_normal(shape)), fmt)
        return q if fmt == "mxfp4" or experts is None else q._replace(tensor_scale=torch.rand(experts, device="cuda"))

    q, q2 = stored(), stored()
    w, image = ops.mx4_pack(q), ops.mx4_pack(q2).image
    at = w.image
    assert ops.mx4_pack(q2, out=w) is w and w.image is at and torch.equal(at, image)
    if fmt == "nvfp4":
        assert torch.equal(w.tensor_scale, q2.tensor_scale.reshape(-1))
    for bad in (q._replace(codes=q.codes[..., :149, :], scales=q.scales[..., :149, :]), ops.mx4_quantize(to_cuda(g.standard_normal((150, 320))), fmt),
                ops.mx4_quantize(to_cuda(g.standard_normal(shape)), "nvfp4" if fmt == "mxfp4" else "mxfp4")):
        with pytest.raises(ValueError, match="out is a packed"):
            ops.mx4_pack(bad, out=w)
    with pytest.raises(ValueError, match="out is a packed"):
        ops.mx4_pack(q, out=w.image)


def test_writes_that_move_no_version_counter_are_seen_after_repack():
    (layer, other), x, want = layers_and_input()
    layer(x)
    layer.codes.data.copy_(other.codes)
    layer.scales.data.copy_(other.scales)
    layer.repack()
    assert torch.equal(layer(x), want[1])
    with torch.inference_mode():
        layer.codes, layer.scales = layer.codes.clone(), layer.scales.clone()
        assert torch.equal(layer(x), want[1])
        layer.codes.zero_()
        layer.repack()
        assert not layer(x).any()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens", [1, 9, 16, 20, 70])
def test_small_values_beside_large_ones(fmt, tokens):
    """A weight row with one value reads one value of x.  In the form for few rows, where bf16 becomes fp16 under a power of two per 256 values,
    it is exact from 2^-32 of the largest of them on, and below off by no more than 2^-40 of it; among more rows it is exact."""
    g = np.random.default_rng(23)
    n = 512
    weight = ops.mx4_pack(ops.mx4_quantize(to_cuda(6.0 * np.eye(n)), fmt, torch.ones(1, device="cuda") if fmt == "nvfp4" else None))
    tops = np.array([2.0 ** e for e in (0, 7, -100, -111, -112, 120)] + [255 * 2.0 ** e for e in (-7, 100, -119)] + [-(2.0 ** -126), 129 * 2.0 ** -7])
    x = np.empty((tokens, n))
    for r in range(tokens):
        for half in (0, 256):
            top = tops[(r + half // 256) % len(tops)]
            v = g.integers(128, 256, 256) * 2.0 ** -8 * 2.0 ** g.integers(-46, 1, 256) * g.choice([-1, 1], 256) * abs(top)
            v[1::16] = 129 * 2.0 ** -7 * 2.0 ** -32 * abs(top)
            v[2::16] = 129 * 2.0 ** -7 * 2.0 ** -33 * abs(top)
            v[::256] = top
            x[r, half:half + 256] = v
    xd = to_cuda(x, torch.bfloat16)
    xv = host(xd).reshape(tokens, 2, 256)
    y = host(ops.mx4_linear(xd, weight, out_dtype=torch.float32)).reshape(tokens, 2, 256)
    top = np.abs(xv).max(-1, keepdims=True)
    err = np.abs(y - 6.0 * xv)
    # (6 x has ten bits: fp32 holds it, from 2^-149 on; the matrix instructions of more rows may take products below 2^-126 as zero)
    few = tokens <= 32
    low = 2.0 ** -149 if few else 2.0 ** -126
    assert np.all(err <= np.where(np.abs(xv) >= 2.0 ** -32 * top, 0.0, 6.0 * 2.0 ** -40 * top if few else 0.0) + low)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens,m", [(1, 200), (16, 200), (32, 130), (40, 200), (250, 200), (1700, 1100)])
@pytest.mark.parametrize("small", [0, -20, -60, -100])
def test_sums_that_stay_in_range(fmt, tokens, m, small):
    """bf16 activations up to the largest there are, weights of any size below one: a sum leaves fp32's range only where the result does.
    Activations times a power of two give the results times that power, bit for bit."""
    g = np.random.default_rng(tokens)
    n = 600
    weight, w = make_weight(g, (m, n), fmt, spread=0.1)
    if small:
        dense = g.standard_normal((m, n)) * np.exp(g.standard_normal((m, 1)) * 0.1) / np.sqrt(n) * 2.0 ** small
        q = ops.mx4_quantize(to_cuda(dense), fmt)
        weight, w = ops.mx4_pack(q), host(ops.mx4_dequantize(q, torch.float32))
    x = to_cuda(g.standard_normal((tokens, n)).clip(-3.9, 3.9), torch.bfloat16)
    up = 125 if small else 122
    y = ops.mx4_linear(x, weight, out_dtype=torch.float32)
    z = ops.mx4_linear(x * 2.0 ** up, weight, out_dtype=torch.float32)
    assert torch.isfinite(z).all()
    check_product(z, host(x * 2.0 ** up), w, torch.float32)
    assert torch.equal(z.double(), y.double() * 2.0 ** up) or small == -100


def test_layer_whose_rows_another_stream_is_writing():
    """The first forward packs what has been enqueued to be written, on whatever stream."""
    (layer, other), x, want = layers_and_input()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        torch.cuda._sleep(DELAY)
        layer.load_state_dict(other.state_dict())
    with torch.cuda.stream(b):
        y = layer(x)
    torch.cuda.synchronize()
    assert torch.equal(y, want[1])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("tokens,m,n", [(2042, 1680, 304), (1921, 1680, 304), (2300, 2500, 640), (1700, 2304, 136), (1537, 3000, 360), (190, 25000, 896)])
def test_tiles_of_an_odd_number_of_steps(fmt, dtype, tokens, m, n):
    """A CTA's second tile behind one of an odd number of steps, with activations that come late (caches emptied in front of every call): the same
    bits every time, and the right ones."""
    g = np.random.default_rng(tokens)
    q = ops.mx4_quantize(to_cuda(g.standard_normal((m, n)) / np.sqrt(n)), fmt)
    weight, w = ops.mx4_pack(q), host(ops.mx4_dequantize(q, torch.float32))
    x = to_cuda(g.standard_normal((tokens, n)), DT[dtype])
    junk = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    first = ops.mx4_linear(x, weight)
    # (dequantised NVFP4 weights are rounded once, by 2^-24 of each)
    check_product(first, host(x), w, DT[dtype])
    for i in range(40):
        junk.fill_(i)
        assert torch.equal(ops.mx4_linear(x, weight), first), i
    ops.check_device_status()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("experts,per,m,n", [(40, 95, 600, 304), (16, 400, 1100, 384), (64, 90, 400, 136)])
def test_experts_tiles_of_an_odd_number_of_steps(fmt, experts, per, m, n):
    g = np.random.default_rng(experts)
    weight, w = make_weight(g, (experts, m, n), fmt)
    counts = g.multinomial(experts * per, g.dirichlet(np.full(experts, 3.0)))
    x = to_cuda(g.standard_normal((int(counts.sum()), n)), torch.bfloat16)
    off = counts_to_offsets(counts)
    junk = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    first = ops.mx4_grouped_linear(x, weight, off)
    at, xv = off.tolist(), host(x)
    for e in range(experts):
        if counts[e]:
            check_product(first[at[e]:at[e + 1]], xv[at[e]:at[e + 1]], w[e], torch.bfloat16)
    for i in range(40):
        junk.fill_(i)
        assert torch.equal(ops.mx4_grouped_linear(x, weight, off), first), i
