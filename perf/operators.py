"""The operators on microscaled 4-bit weights, as cases that can be timed and compared.

Three of them: quantisation there and back (`mx4_quantize`, `mx4_dequantize`), the product of a layer (`mx4_linear`) and the
products grouped by expert with ragged numbers of rows (`mx4_grouped_linear`), in both formats: "mxfp4" (e2m1 values, one
power of two per 32 of them) and "nvfp4" (e2m1 values, one e4m3 scale per 16 of them and one fp32 scale per tensor or expert).
The products take 16-bit activations as they are, or quantise them to the weights' format first (`quantize`).
"""
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
#: borders between neighbouring magnitudes, and whether the border itself belongs to the upper one (ties go to the even code)
BORDERS = ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False))


# ------------------------------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the rows of one token on their way into a 4-bit product or cache: the smallest call, latency alone
        dict(name="quant_mx_1x2048", kind="quant", rows=1, cols=2048, format="mxfp4", dtype="bf16"),
        # the activations of a long prompt in front of the down projection of a larger decoder
        dict(name="quant_mx_2048x14336", kind="quant", rows=2048, cols=14336, format="mxfp4", dtype="bf16"),
        # a weight matrix being quantised, its own scale measured on the way, a width that is no multiple of a block
        dict(name="quant_nv_5376x4100_fp32", kind="quant", rows=5376, cols=4100, format="nvfp4", dtype="fp32"),
        # one attention projection of a small decoder, one token
        dict(name="linear_mx_1tok_2048x2048", kind="linear", m=2048, n=2048, tokens=1, format="mxfp4", dtype="bf16", quantize=False),
        # the widest projection of a larger decoder, a batch of sixteen sequences decoding
        dict(name="linear_nv_16tok_14336x4096", kind="linear", m=14336, n=4096, tokens=16, format="nvfp4", dtype="bf16", quantize=False),
        # a short ragged prompt through a wide-input projection
        dict(name="linear_mx_333tok_2048x11008_fp16", kind="linear", m=2048, n=11008, tokens=333, format="mxfp4", dtype="fp16", quantize=False),
        # a long prompt, activations left in 16 bits
        dict(name="linear_mx_2048tok_14336x4096", kind="linear", m=14336, n=4096, tokens=2048, format="mxfp4", dtype="bf16", quantize=False),
        # a batch of a hundred sequences with 4-bit activations
        dict(name="linear_nv_100tok_4096x4096_q", kind="linear", m=4096, n=4096, tokens=100, format="nvfp4", dtype="fp16", quantize=True),
        # a long prompt with 4-bit activations
        dict(name="linear_mx_2048tok_14336x4096_q", kind="linear", m=14336, n=4096, tokens=2048, format="mxfp4", dtype="bf16", quantize=True),
        # the first projection of 128 experts: 32 decoding sequences with eight experts each, two rows an expert on average
        dict(name="grouped_mx_256rows", kind="grouped", experts=128, m=1536, n=2048, rows=256, behind=0, format="mxfp4", dtype="bf16", quantize=False),
        # the second one with a prompt of 4096 tokens, rows of padding behind the last expert's
        dict(name="grouped_nv_32768rows", kind="grouped", experts=128, m=2048, n=768, rows=32768, behind=37, format="nvfp4", dtype="bf16", quantize=False),
        # the first one with that prompt and 4-bit activations
        dict(name="grouped_mx_32768rows_q", kind="grouped", experts=128, m=1536, n=2048, rows=32768, behind=0, format="mxfp4", dtype="bf16", quantize=True),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    fmt = rng.choice(["mxfp4", "nvfp4"])
    kind = rng.choice(["quant", "linear", "linear", "linear", "grouped", "grouped"])
    if kind == "quant":
        rows, cols = log_int(1, 8192), log_int(32, 14336)
        return dict(kind=kind, rows=rows, cols=cols, format=fmt, dtype=rng.choice(["bf16", "fp16", "fp32"]))
    # widths: mostly whole steps of 64, at times any number
    step = rng.choice([64, 64, 64, 8, 1])
    dtype, quantize = rng.choice(["bf16", "bf16", "fp16"]), rng.random() < 0.4
    if kind == "linear":
        while True:
            tokens = rng.choice([1, rng.randint(2, 16), log_int(1, 128), log_int(17, 2048), log_int(129, 2048)])
            m, n = log_int(64, 14336) // step * step, log_int(64, 14336) // step * step
            if m * n * tokens <= 2048 * 14336 * 4096 and m * n <= 64_000_000:
                return dict(kind=kind, m=m, n=n, tokens=tokens, format=fmt, dtype=dtype, quantize=quantize)
    while True:
        experts, rows = log_int(1, 160), log_int(1, 32768)
        m, n = log_int(64, 4096) // step * step, log_int(64, 4096) // step * step
        if experts * m * n <= 128 * 1536 * 2048 and rows * m * n <= 32768 * 1536 * 2048:
            return dict(kind=kind, experts=experts, m=m, n=n, rows=rows, behind=rng.choice([0, 0, log_int(1, 200)]), format=fmt, dtype=dtype, quantize=quantize)


def _block(fmt):
    return 32 if fmt == "mxfp4" else 16


def _weight_bytes(m, n, fmt):
    return m * ((n + 1) // 2 + -(-n // _block(fmt)))


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "quant":
        values = case["rows"] * case["cols"]
        held = _weight_bytes(case["rows"], case["cols"], case["format"])
        return {"bytes": 2 * values * size + 2 * held, "flops": 0}
    m, n = case["m"], case["n"]
    if case["kind"] == "linear":
        t = case["tokens"]
        return {"bytes": _weight_bytes(m, n, case["format"]) + t * (m + n) * size, "flops": 2 * t * m * n}
    r, e = case["rows"], case["experts"]
    touched = e * (1 - (1 - 1 / e) ** r)
    return {"bytes": touched * _weight_bytes(m, n, case["format"]) + (r * (m + n) + case["behind"] * m) * size, "flops": 2 * r * m * n}


# ------------------------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------------------------
def _blocks_of(x, fmt):
    """x (..., n) in 64 bits as (..., blocks, block), zeros behind the last value."""
    b = _block(fmt)
    pad = -x.shape[-1] % b
    x = x.double()
    if pad:
        x = torch.nn.functional.pad(x, (0, pad))
    return x.unflatten(-1, (-1, b))


def _tensor_scale(x):
    """The fp32 scale that puts the largest value at the top of both 4-bit levels."""
    return torch.clamp(x.float().abs().amax() / 2688.0, min=2.0 ** -126).reshape(1)


def _round_e4m3(v):
    """64-bit values >= 0 to the nearest e4m3 value, ties to even, largest 448."""
    v = v.clamp(max=448.0)
    _, e = torch.frexp(v)
    quantum = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return (torch.round(v / quantum) * quantum).clamp(max=448.0)


def _quantize(x, fmt, tensor_scale=None):
    """(codes 0..15 of every value, padded to whole blocks; the scale of every block as a number; its byte)."""
    xb = _blocks_of(x, fmt)
    amax = xb.abs().amax(-1)
    if fmt == "mxfp4":
        _, e = torch.frexp(amax)
        power = torch.where(amax > 0, (e - 3).clamp(-127, 125), -127)
        scale, byte = torch.exp2(power.double()), (power + 127).to(torch.uint8)
        step = scale
    else:
        t = tensor_scale.double()
        scale = _round_e4m3(amax / (6.0 * t))
        byte = scale.float().to(torch.float8_e4m3fn).view(torch.uint8)
        step = scale * t
    q = xb.abs() / torch.where(step > 0, step, 1.0).unsqueeze(-1)
    q = torch.where((step > 0).unsqueeze(-1), q, 0.0)
    code = torch.zeros_like(q, dtype=torch.uint8)
    code += (q > 0.25).to(torch.uint8) + (q >= 0.75).to(torch.uint8) + (q > 1.25).to(torch.uint8) + (q >= 1.75).to(torch.uint8)
    code += (q > 2.5).to(torch.uint8) + (q >= 3.5).to(torch.uint8) + (q > 5.0).to(torch.uint8)
    code += torch.signbit(xb).to(torch.uint8) * 8
    return code, scale, byte


def _values(code, scale, n, tensor_scale=None):
    """What codes and scales stand for, (..., n) in 32 bits."""
    table = torch.tensor(MAGNITUDES + tuple(-v for v in MAGNITUDES), dtype=torch.float32, device=code.device)
    v = table[code.long()] * scale.float().unsqueeze(-1)
    if tensor_scale is not None:
        v = v * tensor_scale.float().reshape(-1, *[1] * (v.dim() - 1))
    return v.flatten(-2)[..., :n]


def _quantized(x, fmt):
    """x as its 4-bit form has it, in 32 bits."""
    t = _tensor_scale(x) if fmt == "nvfp4" else None
    code, scale, _ = _quantize(x, fmt, t)
    return _values(code, scale, x.shape[-1], t)


def _unpacked(codes, scales, n, fmt, tensor_scale):
    """Stored bytes as values, (..., n) in 32 bits."""
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    b = _block(fmt)
    code = torch.nn.functional.pad(code, (0, scales.shape[-1] * b - code.shape[-1])).unflatten(-1, (-1, b))
    scale = torch.exp2(scales.float() - 127.0) if fmt == "mxfp4" else scales.view(torch.float8_e4m3fn).float()
    return _values(code, scale, n, tensor_scale)


def _plain_linear(s):
    x = _quantized(s["x"], s["format"]) if s["quantize"] else s["x"].float()
    w = _unpacked(s["codes"], s["scales"], s["n"], s["format"], s["tensor_scale"])
    return (x @ w.t()).to(s["x"].dtype)


def _plain_grouped(s):
    """Every expert's rows in a matrix of as many rows as the largest expert has, one batched product, and back."""
    offsets, x = s["offsets"].long(), s["x"]
    used = s["used"]
    x = _quantized(x[:used], s["format"]) if s["quantize"] else x[:used].float()
    row = torch.arange(used, device=x.device)
    expert = torch.searchsorted(offsets[1:], row, right=True)
    place = row - offsets[expert]
    padded = x.new_zeros(s["experts"], s["most"], s["n"])
    padded[expert, place] = x
    w = _unpacked(s["codes"], s["scales"], s["n"], s["format"], s["tensor_scale"])
    y = torch.bmm(padded, w.transpose(1, 2))
    out = torch.zeros(s["x"].shape[0], w.shape[1], dtype=s["x"].dtype, device=x.device)
    out[:used] = y[expert, place].to(out.dtype)
    return out


# ------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _stored(g, shape, fmt):
    """A seeded weight matrix (or one per expert) as a checkpoint holds it: codes two to a byte, scales, fp32 scale(s)."""
    experts = shape[0] if len(shape) == 3 else None
    n = shape[-1]
    codes, scales, ts = [], [], []
    for _ in range(experts or 1):
        w = torch.randn(shape[-2:], generator=g, device="cuda") * (0.7 / n ** 0.5)
        t = _tensor_scale(w) if fmt == "nvfp4" else None
        code, _, byte = _quantize(w, fmt, t)
        code = code.flatten(-2)[:, :n + n % 2]
        if n % 2:
            code[:, n] = 0
        codes.append(code[:, 0::2] | (code[:, 1::2] << 4))
        scales.append(byte)
        ts.append(t)
    if experts is None:
        return codes[0].contiguous(), scales[0].contiguous(), ts[0]
    return torch.stack(codes), torch.stack(scales), torch.cat(ts) if fmt == "nvfp4" else None


def _activations(g, rows, cols, dtype):
    """Normal values with a few channels that stand out, as the inputs of a decoder's projections have them."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= torch.where(torch.rand(cols, generator=g, device="cuda") < 0.01, 8.0, 1.0)
    return x.to(DTYPES[dtype])


def _inputs(case, seed):
    g, fmt = _gen(seed), case["format"]
    if case["kind"] == "quant":
        return dict(kind="quant", format=fmt, x=_activations(g, case["rows"], case["cols"], case["dtype"]))
    m, n = case["m"], case["n"]
    s = dict(kind=case["kind"], format=fmt, n=n, quantize=case["quantize"])
    if case["kind"] == "linear":
        s["codes"], s["scales"], s["tensor_scale"] = _stored(g, (m, n), fmt)
        s["x"] = _activations(g, case["tokens"], n, case["dtype"])
        return s
    e, rows = case["experts"], case["rows"]
    s["codes"], s["scales"], s["tensor_scale"] = _stored(g, (e, m, n), fmt)
    s["x"] = _activations(g, rows + case["behind"], n, case["dtype"])
    chosen = torch.randint(0, e, (rows,), generator=g, device="cuda")
    counts = torch.bincount(chosen, minlength=e)
    s["offsets"] = torch.cat((counts.new_zeros(1), counts.cumsum(0))).to(torch.int32)
    s["experts"], s["used"], s["most"] = e, rows, int(counts.max())
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and s["kind"] != "quant":
        from glq_b200 import ops
        # the weights as a program keeps them: laid out once when they are loaded
        s["weight"] = ops.mx4_pack(ops.Mx4Tensor(s["codes"], s["scales"], s["format"], s["n"], s["tensor_scale"]))
    return s


def run(state):
    if own:
        from glq_b200 import ops
        if state["kind"] == "quant":
            return ops.mx4_dequantize(ops.mx4_quantize(state["x"], state["format"]), state["x"].dtype)
        if state["kind"] == "linear":
            return ops.mx4_linear(state["x"], state["weight"], quantize_input=state["quantize"])
        return ops.mx4_grouped_linear(state["x"], state["weight"], state["offsets"], quantize_input=state["quantize"])
    if state["kind"] == "quant":
        return _quantized(state["x"], state["format"]).to(state["x"].dtype)
    return _plain_linear(state) if state["kind"] == "linear" else _plain_grouped(state)


# ------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits, apart from the plain forms
# ------------------------------------------------------------------------------------------------------------------
def _nearest(q):
    """Real numbers >= 0 to the nearest e2m1 magnitude: a search over the borders, a number on one goes to its even neighbour."""
    borders = torch.tensor([b for b, _ in BORDERS], dtype=torch.float64, device=q.device)
    upper = torch.tensor([u for _, u in BORDERS] + [False], device=q.device)
    at = torch.bucketize(q.contiguous(), borders)
    on = (at < 7) & (q == borders[at.clamp(max=6)])
    return torch.tensor(MAGNITUDES, dtype=torch.float64, device=q.device)[at + (on & upper[at]).long()]


def _exact_quantized(x, fmt):
    x64, n, b = x.double(), x.shape[-1], _block(fmt)
    out = torch.empty_like(x64)
    whole = n // b * b
    t = max(float((x.abs().amax().float() / 2688.0)), 2.0 ** -126)
    for lo, hi in ((0, whole), (whole, n)):
        if lo == hi:
            continue
        v = x64[..., lo:hi]
        v = v.reshape(*v.shape[:-1], -1, b) if hi == whole else v.unsqueeze(-2)
        top = v.abs().max(-1, keepdim=True).values
        if fmt == "mxfp4":
            # (the logarithm of a value just below a power of two may round up to it: compared with the power itself)
            e = torch.floor(torch.log2(top.clamp(min=2.0 ** -200)))
            e = torch.where(torch.exp2(e) > top, e - 1, e)
            e = torch.where(torch.exp2(e + 1) <= top, e + 1, e)
            step = torch.exp2((e - 2).clamp(-127, 125))
        else:
            levels = torch.arange(127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
            ratio = (top / (6.0 * t)).clamp(max=448.0)
            middle = (levels[1:] + levels[:-1]) / 2
            at = torch.bucketize(ratio.contiguous(), middle)
            on = (at < 126) & (ratio == middle[at.clamp(max=125)])
            step = levels[at + (on & (at % 2 == 1)).long()] * t
        safe = torch.where(step > 0, step, 1.0)
        r = torch.where(step > 0, _nearest(v.abs() / safe) * step, 0.0) * torch.sign(v)
        out[..., lo:hi] = r.flatten(-2)
    return out


def _exact_weights(codes, scales, n, fmt, tensor_scale):
    table = torch.tensor(MAGNITUDES, dtype=torch.float64, device=codes.device)
    out = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.float64, device=codes.device)
    out[..., 0::2] = table[(codes & 7).long()] * (1 - 2 * ((codes >> 3) & 1).double())
    out[..., 1::2] = table[((codes >> 4) & 7).long()] * (1 - 2 * (codes >> 7).double())
    scale = 2.0 ** (scales.double() - 127) if fmt == "mxfp4" else scales.view(torch.float8_e4m3fn).double() * tensor_scale.double()
    return out[..., :n] * scale.repeat_interleave(_block(fmt), -1)[..., :n]


def exact(case, seed):
    s = _inputs(case, seed)
    fmt, x = s["format"], s["x"]
    if s["kind"] == "quant":
        return _exact_quantized(x, fmt)
    if s["kind"] == "linear":
        x = _exact_quantized(x, fmt) if s["quantize"] else x.double()
        return x @ _exact_weights(s["codes"], s["scales"], s["n"], fmt, s["tensor_scale"]).t()
    at = s["offsets"].tolist()
    out = torch.zeros(x.shape[0], case["m"], dtype=torch.float64, device=x.device)
    x = _exact_quantized(x[:s["used"]], fmt) if s["quantize"] else x.double()
    for e in range(s["experts"]):
        if at[e] < at[e + 1]:
            w = _exact_weights(s["codes"][e], s["scales"][e], s["n"], fmt, s["tensor_scale"][e] if fmt == "nvfp4" else None)
            out[at[e]:at[e + 1]] = x[at[e]:at[e + 1]] @ w.t()
    return out
