"""Microscaled 4-bit floating point without a GPU: the oracle against itself, the ABI's structure, the refusals."""
import ctypes
import os
import re
import subprocess
import sys

import numpy as np
import pytest
import torch

import mx4_oracle as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_oracle_rounds_to_the_nearest_value_and_to_even_codes():
    x = np.array([[0.0, 0.25, 0.26, 0.74, 0.75, 1.25, 1.75, 2.5, 2.6, 3.5, 5.0, 5.01, 6.0, -0.25, -5.0, 4.0]])
    code, byte = O.quantize(x, "nvfp4", 1.0)
    assert byte.tolist() == [[56]]                              # 6 / 6 = 1.0 in e4m3
    assert O.MAGNITUDES[code & 7].tolist() == [[0, 0, 0.5, 0.5, 1, 1, 2, 2, 3, 4, 4, 6, 6, 0, 4, 4]]
    code, byte = O.quantize(np.array([[7.9, 4.0, -0.5] + [0.0] * 29]), "mxfp4")
    assert byte.tolist() == [[127]] and O.values(code, byte, "mxfp4")[0, :3].tolist() == [6.0, 4.0, -0.5]
    assert O.quantize(np.zeros((1, 32)), "mxfp4")[1].tolist() == [[0]]
    assert O.quantize(np.full((1, 32), np.inf), "mxfp4")[1].tolist() == [[255]]


def test_oracle_nibbles_round_trip():
    code = np.random.default_rng(0).integers(0, 16, (3, 7), dtype=np.uint8)
    assert np.array_equal(O.unpack_nibbles(O.pack_nibbles(code), 7), code)


def test_e4m3_table_is_torchs():
    assert np.array_equal(torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy(), O.E4M3)


@pytest.fixture(scope="module")
def lib():
    from glq_b200 import _lib, build
    build.build()
    return _lib.load()


def test_struct_layout_matches_header(tmp_path):
    from glq_b200 import _lib
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "glq_b200.h"\nint main(){printf("%zu %zu %zu %zu\\n", sizeof(GlqbMx4Weight),'
                   '__builtin_offsetof(GlqbMx4Weight, tensor_scale), __builtin_offsetof(GlqbMx4Weight, format), __builtin_offsetof(GlqbMx4Weight, n));}')
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    D = _lib.Mx4WeightDesc
    assert out == [ctypes.sizeof(D), D.tensor_scale.offset, D.format.offset, D.n.offset]


def test_image_sizes(lib):
    # tiles of 128 x 256: 16 KiB of codes and 1 (blocks of 32) or 2 KiB (of 16) of scales, MXFP4 two bytes per row behind them
    assert lib.glqb_mx4_image_bytes(0, 1, 128, 256) == 16384 + 1024 + 256
    assert lib.glqb_mx4_image_bytes(1, 1, 128, 256) == 16384 + 2048
    assert lib.glqb_mx4_image_bytes(1, 5, 129, 257) == 5 * 4 * (16384 + 2048)
    assert lib.glqb_mx4_image_bytes(2, 1, 128, 256) == 0 and lib.glqb_mx4_image_bytes(0, 0, 128, 256) == 0


def test_c_entries_refuse_before_any_cuda_call(lib):
    from glq_b200 import _lib
    p = 4096                                                    # never dereferenced: each call is refused

    def refused(rc, code, text):
        assert rc == code and text in lib.glqb_last_error().decode(), (rc, lib.glqb_last_error())

    refused(lib.glqb_mx4_quantize(p, 0, 32, 1, 32, 2, None, None, p, p, None), -1, "format")
    refused(lib.glqb_mx4_quantize(p, 3, 32, 1, 32, 0, None, None, p, p, None), -1, "dtype")
    refused(lib.glqb_mx4_quantize(p, 0, 32, -1, 32, 0, None, None, p, p, None), -1, "-1 x 32")
    refused(lib.glqb_mx4_quantize(p, 0, 31, 2, 32, 0, None, None, p, p, None), -1, "apart")
    refused(lib.glqb_mx4_quantize(p, 0, 32, 1, 32, 1, None, None, p, p, None), -1, "tensor_scale")
    refused(lib.glqb_mx4_quantize(None, 0, 32, 1, 32, 0, None, None, p, p, None), -1, "null")
    assert lib.glqb_mx4_quantize(None, 0, 32, 0, 32, 0, None, None, None, None, None) == 0
    refused(lib.glqb_mx4_dequantize(p, p, None, 1, 1, 32, 1, p, 0, None), -1, "tensor_scale")
    refused(lib.glqb_mx4_dequantize(p, p, None, 1, 1, 32, 0, p, 7, None), -1, "dtype")
    refused(lib.glqb_mx4_pack(p, p, 0, 1, 0, 32, p, None), -1, "1 x 0 x 32")
    refused(lib.glqb_mx4_pack(p, p, 0, 1, 32, 32, p + 64, None), -1, "aligned")
    refused(lib.glqb_mx4_pack(p, p, 0, 65536, 65536, 65536, p, None), -1, "tiles")

    def product(w, x=p, xd=1, xs=64, rows=2, offsets=None, q=0, y=p, yd=1, ys=64, ws=None, size=0, xscale=None):
        return lib.glqb_mx4_product(ctypes.byref(w), x, xd, xs, rows, offsets, 0, q, xscale, y, yd, ys, 0, 0, ws, size, None)

    w = _lib.Mx4WeightDesc(p, None, 0, 1, 64, 64)
    refused(product(_lib.Mx4WeightDesc(p, None, 5, 1, 64, 64)), -1, "format")
    refused(product(_lib.Mx4WeightDesc(p, None, 0, 2, 64, 64)), -1, "offsets")
    refused(product(_lib.Mx4WeightDesc(p, None, 1, 1, 64, 64)), -1, "null")
    refused(product(w, xd=2), -1, "fp32")
    refused(product(w, yd=4), -1, "dtype")
    refused(product(w, rows=1 << 31), -1, "rows")
    refused(product(w, xs=63), -1, "overlap")
    refused(product(w, ys=63), -1, "overlap")
    refused(product(w, y=None), -1, "null")
    refused(product(w, q=1), -3, "workspace")
    assert product(w, rows=0) == 0


def test_operators_refuse_host_tensors_and_wrong_arguments():
    from glq_b200 import ops
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.mx4_quantize(x)
    with pytest.raises(ValueError, match="mxfp4"):
        ops.mx4_quantize(x, "fp4")
    q = ops.Mx4Tensor(torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8), "mxfp4", 64)
    for call in (ops.mx4_dequantize, ops.mx4_pack):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call(q)
    with pytest.raises(ValueError, match="mx4_pack"):
        ops.mx4_linear(x, q)
    with pytest.raises(ValueError, match="mx4_pack"):
        ops.mx4_grouped_linear(x, q, torch.zeros(3, dtype=torch.int32))


def test_sizes_beyond_what_is_counted_are_refused(lib):
    from glq_b200 import _lib
    p, big = 4096, (1 << 30) + 1

    def product(w, rows, offsets=None, stride=1 << 40):
        return lib.glqb_mx4_product(ctypes.byref(w), p, 1, stride, rows, offsets, 0, 0, None, p, 1, stride, 0, 0, None, 0, None), lib.glqb_last_error().decode()

    for w, rows, offsets, text in ((_lib.Mx4WeightDesc(p, None, 0, 1025, 64, 64), 2, p, "at most 1024"),
                                   (_lib.Mx4WeightDesc(p, None, 0, 1, big, 64), 2, None, str(big)),
                                   (_lib.Mx4WeightDesc(p, None, 0, 1, 64, big), 2, None, str(big)),
                                   (_lib.Mx4WeightDesc(p, None, 0, 1, 64, 64), 0x7FFF0001, None, "rows"),
                                   (_lib.Mx4WeightDesc(p, None, 0, 1, 1 << 20, 64), 1 << 18, None, "too many")):
        rc, said = product(w, rows, offsets)
        assert rc == -1 and text in said, said
        assert lib.glqb_mx4_workspace_bytes(ctypes.byref(w), rows, 1 << 40, p, 1) == 0
    two = _lib.Mx4WeightDesc(p, None, 0, 2, 64, 64)
    assert lib.glqb_mx4_workspace_bytes(ctypes.byref(two), 0x7FFF0000, 64, p, 1) == 0 and product(two, 0x7FFF0000, p)[0] == -1
    assert lib.glqb_mx4_workspace_bytes(ctypes.byref(two), 1000, 64, p, 1) > 1000 * 32
    for m, n in ((big, 1), (1, big)):
        assert lib.glqb_mx4_pack(p, p, 0, 1, m, n, p, None) == -1
    assert lib.glqb_mx4_pack(p, p, 0, 1025, 8, 8, p, None) == -1 and "1024 experts" in lib.glqb_last_error().decode()
    assert lib.glqb_mx4_pack(p, p, 0, 1024, 1 << 26, 1, p, None) == -1


def test_layer_of_4_bit_weights_on_the_host():
    from glq_b200.linear import Mx4Linear
    layer = Mx4Linear(50, 33, bias=True, format="nvfp4")
    shapes = {k: (tuple(v.shape), v.dtype) for k, v in layer.state_dict().items()}
    assert shapes == {"codes": ((33, 25), torch.uint8), "scales": ((33, 4), torch.uint8), "tensor_scale": ((1,), torch.float32),
                      "bias": ((33,), torch.float32)}
    layer.half()
    assert layer.tensor_scale.dtype == layer.bias.dtype == torch.float32 and layer.codes.dtype == torch.uint8
    layer.load_state_dict({**layer.state_dict(), "tensor_scale": torch.full((1,), 0.25)})
    assert layer.tensor_scale.item() == 0.25
    assert set(Mx4Linear(64, 8).state_dict()) == {"codes", "scales"}
    with pytest.raises(RuntimeError, match="no CPU path"):
        layer(torch.zeros(1, 50))
    with pytest.raises(ValueError, match="mxfp4"):
        Mx4Linear(8, 8, format="fp4")


def test_layer_waits_for_its_packing_and_for_its_readers(monkeypatch):
    """Whoever is given the packed weight finds it complete, whatever stream they run on; a weight that is packed again goes when nothing
    reads it any more.  (The order of the host's calls, without a GPU.)"""
    import contextlib
    import types
    from glq_b200 import linear
    calls = []

    def pack(rows, out=None):
        calls.append("pack")
        return types.SimpleNamespace(image=types.SimpleNamespace(device="device"), tensor_scale=None)

    monkeypatch.setattr(linear.ops, "mx4_pack", pack)
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: types.SimpleNamespace(synchronize=lambda: calls.append("wait"), cuda_stream=7))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: calls.append("all"))
    layer = linear.Mx4Linear(64, 8)
    first = layer.weight
    assert calls == ["pack", "wait"] and layer.weight is first and calls == ["pack", "wait"]
    for change in (lambda: layer.codes.add_(1), layer.half, layer.repack, lambda: layer.load_state_dict(layer.state_dict())):
        calls.clear()
        change()
        assert layer.weight is not None
        assert calls == ["all", "pack", "wait"], calls


def test_layer_keeps_the_memory_of_its_packed_weight(monkeypatch):
    """A captured graph holds the address of the packed weight: packed again, a layer offers the old one's memory, unless it has
    gone to another device.  (The host's calls, without a GPU.)"""
    import contextlib
    import types
    from glq_b200 import linear
    offered = []

    def pack(rows, out=None):
        offered.append(out)
        return out or types.SimpleNamespace(image=types.SimpleNamespace(device=rows.codes.device), tensor_scale=None, _holds=lambda rows: rows.cols == 64)

    monkeypatch.setattr(linear.ops, "mx4_pack", pack)
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: types.SimpleNamespace(synchronize=lambda: None, cuda_stream=7))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    layer = linear.Mx4Linear(64, 8)
    first = layer.weight
    for change in (lambda: layer.codes.add_(1), layer.half, layer.repack, lambda: layer.load_state_dict(layer.state_dict(), assign=True)):
        change()
        assert layer.weight is first and offered[-1] is first
    layer.to("meta")
    assert layer.weight is not first and offered[-1] is None


def _source(name):
    """C++ source without comments, and without the semicolons of loop heads and strings in calls."""
    with open(os.path.join(ROOT, "glq_b200", "csrc", name)) as f:
        text, depth, out = "\n".join(line.split("//")[0] for line in f.read().split("\n")), 0, []
    for c in text:
        depth += (c == "(") - (c == ")")
        out.append(" " if c == ";" and depth else c)
    return "".join(out)


def _blocks_around(text, at):
    """What stands in front of every brace that is open at a place of C++ source: the conditions and loops it is under."""
    heads, depth = [], 0
    for i in range(at, -1, -1):
        if text[i] == "}":
            depth += 1
        elif text[i] == "{":
            if depth:
                depth -= 1
            else:
                start = max(text.rfind(c, 0, i) for c in ";{}")
                heads.append(text[start + 1:i])
    return heads


def test_whole_warps_wait_with_one_outcome():
    """A bounded wait gives up lane by lane.  Where it is a warp's, whose lanes go on to votes and matrix instructions together, either
    its outcome is one for all of them, or no lane leaves its place by it; a wait that ends a loop is for blocks that a single lane runs."""
    seen = 0
    for name in ("glqb_mx4_gemm.cu", "glqb_mx4_mv.cu"):
        text = _source(name)
        at = text.find("mbar_wait(")
        while at >= 0:
            start = max(text.rfind(c, 0, at) for c in ";{}")
            heads = [text[start + 1:at]] + _blocks_around(text, at)
            line = text[at:text.find("\n", at)]
            stays = not re.search(r"\b(break|continue|return)\b", line) and not any(re.search(r"\bok\b", h) for h in heads[1:])
            assert stays or any("lane == 0" in h or "elect_one()" in h for h in heads), f"{name}: {text[at:at + 60]}"
            seen += 1
            at = text.find("mbar_wait(", at + 1)
    assert seen >= 6


def test_instructions_of_whole_warps_are_reached_by_whole_warps():
    """Cluster barriers gather their warp first; the loops that read tensor memory have no exit for single lanes, and lanes that store nothing
    meet the others in front of the next read."""
    text = {name: _source(name) for name in ("glqb_mx4_gemm.cu", "glqb_mx4_gemm.cuh", "glqb_mx4_mv.cu")}
    seen = 0
    for name, source in text.items():
        for m in re.finditer(r"barrier\.cluster", source):
            start = source.rfind("{", 0, m.start())
            assert "__syncwarp" in source[start:m.start()], f"{name}: {source[m.start() - 80:m.start() + 60]}"
            seen += 1
    assert seen >= 4
    gemm = text["glqb_mx4_gemm.cu"]
    for name in ("drain_wide", "drain_tile"):
        at = gemm.index(f"void {name}(")
        body = gemm[at:gemm.index("template <", at)]
        assert "tmem_ld" in body and "continue" not in body and "break" not in body
    narrow = body[body.rindex("tmem_ld8"):]
    assert narrow.index("mx4_put") < narrow.index("__syncwarp")
    alloc = gemm[gemm.index("void alloc_all("):gemm.index("void dealloc_all(")]
    assert alloc.index("__syncwarp") < alloc.index("tcgen05.alloc")


def test_modules_import_without_torchs_cuda_names():
    """The host logic (checkpoints, loading, layers' buffers) is there with a build of torch that has no CUDA."""
    code = ("import torch\n"
            "for name in [n for n in dir(torch._C) if n.startswith('_cuda_')]:\n"
            "    delattr(torch._C, name)\n"
            "import glq_b200, glq_b200.ops, glq_b200.linear, glq_b200.loader, glq_b200.dropin, glq_b200.checkpoint\n"
            "from glq_b200.linear import Mx4Linear\n"
            "assert set(Mx4Linear(64, 8).state_dict()) == {'codes', 'scales'}\n")
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr


def test_addresses_that_kernels_cannot_use_are_refused(lib):
    """Before any CUDA call: an image or workspace that bulk copies cannot read, values that lie between their places."""
    from glq_b200 import _lib
    p = 1 << 20                                                 # never dereferenced: each call is refused

    def refused(rc, text):
        assert rc == -1 and text in lib.glqb_last_error().decode(), (rc, lib.glqb_last_error())

    def product(w, x=p, xd=1, offsets=None, wide=0, q=0, xscale=None, y=p, yd=1, ws=None, size=0):
        return lib.glqb_mx4_product(ctypes.byref(w), x, xd, 64, 40, offsets, wide, q, xscale, y, yd, 64, 0, 0, ws, size, None)

    mx, nv = _lib.Mx4WeightDesc(p, None, 0, 1, 64, 64), _lib.Mx4WeightDesc(p, p, 1, 1, 64, 64)
    for off in (16, 64, 1):
        refused(product(_lib.Mx4WeightDesc(p + off, None, 0, 1, 64, 64)), "128-byte aligned")
    for off in (1, 4, 8):
        refused(product(mx, q=1, ws=p + off, size=1 << 20), "16-byte aligned")
    for call in (lambda: product(mx, x=p + 1), lambda: product(mx, x=p + 2, xd=2, q=1, ws=p, size=1 << 20), lambda: product(mx, y=p + 1),
                 lambda: product(mx, y=p + 2, yd=2), lambda: product(mx, offsets=p + 2), lambda: product(mx, offsets=p + 4, wide=1),
                 lambda: product(_lib.Mx4WeightDesc(p, p + 2, 1, 1, 64, 64)), lambda: product(nv, q=1, xscale=p + 1, ws=p, size=1 << 20),
                 lambda: lib.glqb_mx4_quantize(p + 1, 0, 32, 1, 32, 0, None, None, p, p, None),
                 lambda: lib.glqb_mx4_quantize(p + 2, 2, 32, 1, 32, 0, None, None, p, p, None),
                 lambda: lib.glqb_mx4_quantize(p, 0, 32, 1, 32, 1, p + 2, None, p, p, None),
                 lambda: lib.glqb_mx4_quantize(p, 0, 32, 1, 32, 1, None, p + 1, p, p, None),
                 lambda: lib.glqb_mx4_dequantize(p, p, None, 1, 1, 32, 0, p + 1, 0, None),
                 lambda: lib.glqb_mx4_dequantize(p, p, p + 1, 1, 1, 32, 1, p, 0, None)):
        refused(call(), "not aligned")


def test_rows_too_long_to_be_counted_are_refused(monkeypatch):
    """Sizes pass a C interface of 32 bits, which would cut 2^32 + 32 values to 32 without a word.  (On tensors without memory.)"""
    from glq_b200 import mx4, ops
    monkeypatch.setattr(mx4, "_cuda", lambda t, name: None)
    monkeypatch.setattr(mx4, "_call", lambda *a: pytest.fail("a call was made"))
    for n in (2 ** 31, 2 ** 32 + 32):
        with pytest.raises(ValueError, match="at most 2147483647"):
            ops.mx4_quantize(torch.empty(n, dtype=torch.bfloat16, device="meta"))
        q = ops.Mx4Tensor(torch.empty(1, n // 2, dtype=torch.uint8, device="meta"), torch.empty(1, n // 32, dtype=torch.uint8, device="meta"), "mxfp4", n)
        for call in (ops.mx4_dequantize, ops.mx4_pack):
            with pytest.raises(ValueError, match="at most 2147483647"):
                call(q)
        for lead in ((n,), (n, 1)):
            q = ops.Mx4Tensor(torch.empty(*lead, 16, dtype=torch.uint8, device="meta"), torch.empty(*lead, 1, dtype=torch.uint8, device="meta"), "mxfp4", 32)
            with pytest.raises(ValueError, match="at most 2147483647"):
                ops.mx4_pack(q)


def test_layer_on_the_host_has_no_packed_weight():
    from glq_b200.linear import Mx4Linear
    with pytest.raises(RuntimeError, match="codes must be a CUDA tensor"):
        Mx4Linear(64, 8).weight


@pytest.mark.parametrize("assign", [False, True])
def test_layer_loads_bytes_of_any_one_byte_type(assign):
    """Checkpoints give scales (and codes) types of their own; their bytes are what counts."""
    from glq_b200.linear import Mx4Linear
    g = np.random.default_rng(0)
    for fmt, dtypes in (("nvfp4", (torch.uint8, torch.float8_e4m3fn, torch.int8)), ("mxfp4", (torch.uint8, torch.float8_e8m0fnu, torch.int8))):
        scales = torch.from_numpy(g.integers(0, 127, (8, 64 // O.BLOCK[fmt]), dtype=np.uint8))
        codes = torch.from_numpy(g.integers(0, 256, (8, 32), dtype=np.uint8))
        for dtype in dtypes:
            layer = Mx4Linear(64, 8, format=fmt)
            state = {"codes": codes.view(torch.int8) if dtype == torch.int8 else codes, "scales": scales.view(dtype)}
            if fmt == "nvfp4":
                state["tensor_scale"] = torch.tensor(0.25)
            kept = dict(state)
            layer.load_state_dict(state, assign=assign)
            assert layer.scales.dtype == layer.codes.dtype == torch.uint8
            assert torch.equal(layer.scales, scales) and torch.equal(layer.codes, codes)
            assert all(state[k] is kept[k] for k in kept)
            if fmt == "nvfp4":
                assert layer.tensor_scale.shape == (1,) and layer.tensor_scale.item() == 0.25
        with pytest.raises(RuntimeError, match="scales holds torch.float32"):
            Mx4Linear(64, 8, format=fmt).load_state_dict({"codes": codes, "scales": scales.float()}, strict=False)
        with pytest.raises(RuntimeError, match="scales holds torch.float32"):
            torch.nn.Sequential(Mx4Linear(64, 8, format=fmt)).load_state_dict({"0.codes": codes, "0.scales": scales.float()}, strict=False)


def test_layer_of_a_dense_weight_has_its_own_bias(monkeypatch):
    """Loading into the layer must not write to the bias that it was made from."""
    from glq_b200 import linear
    monkeypatch.setattr(linear.ops, "mx4_quantize", lambda w, fmt: linear.ops.Mx4Tensor(torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8), fmt, 64))
    bias = torch.nn.Parameter(torch.arange(8.0))
    layer = linear.Mx4Linear.from_weight(torch.zeros(8, 64), bias)
    layer.load_state_dict({**layer.state_dict(), "bias": torch.ones(8)})
    assert torch.equal(bias.detach(), torch.arange(8.0)) and torch.equal(layer.bias, torch.ones(8)) and not layer.bias.requires_grad


def test_layer_packs_behind_writes_on_other_streams(monkeypatch):
    """What the first forward packs is kept: rows that another stream is still writing are waited for.  (The host's calls, without a GPU.)"""
    import contextlib
    import types
    from glq_b200 import linear
    calls = []

    class Rows:
        is_cuda, device, _version = True, torch.device("cuda:0"), 0
        get_device = staticmethod(lambda: 0)
        is_inference = staticmethod(lambda: False)

    def pack(rows, out=None):
        calls.append("pack")
        return types.SimpleNamespace(image=types.SimpleNamespace(device=rows.codes.device), tensor_scale=None, _holds=lambda rows: True)

    monkeypatch.setattr(linear.ops, "mx4_pack", pack)
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: types.SimpleNamespace(synchronize=lambda: calls.append("wait"), cuda_stream=7))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device: calls.append(str(device)))
    layer = linear.Mx4Linear(64, 8)
    del layer.codes, layer.scales
    layer.codes, layer.scales = Rows(), Rows()
    for _ in range(2):
        assert layer.weight is layer.weight
        assert calls == ["cuda:0", "pack", "wait"]
        calls.clear()
        layer.repack()


def _ring_is_safe(stages, steps, tiles, alternate):
    """Two groups of warps fill a ring of `stages` in turn, one thread empties it in order.  A group waits for the round before by parity, which
    a barrier two rounds behind answers with yes: the round before that must be known to be over, by what the group waited for last.
    `alternate`: a group's steps are two apart over the tiles' borders; else each tile begins with the first group."""
    for group in (0, 1):
        over, g0 = -1, 0                                        # the last step known to be read (steps are read in order)
        mine = group
        for _ in range(tiles):
            for k in range(mine, steps, 2):
                g = g0 + k
                if g - 2 * stages > over:
                    return False
                over = max(over, g - stages)
            g0 += steps
            if alternate:
                mine ^= steps & 1
    return True


def test_groups_that_fill_a_ring_stay_within_what_parity_can_tell():
    for steps in range(1, 12):
        for stages in (2, 3, 4):                                # what two accumulators of up to 192, 160 and 128 columns leave
            assert _ring_is_safe(stages, steps, 9, True)
            assert _ring_is_safe(stages, steps, 9, False) == (stages > 2 or steps % 2 == 0 or steps == 1)
    text = _source("glqb_mx4_gemm.cu")
    loop = text[text.index("int mine = group"):]
    assert re.search(r"for \(int k = mine  k < steps \+ mine  k \+= 2", loop) and re.search(r"mine \^= steps & 1;", loop)
    assert "a.add(group, R.a_stages)" in text and "a.add(2, R.a_stages)" in loop and ".back(" not in text
    assert "std::min(4, (512 - 2 * R.acc_cols) / 64)" in text.replace(" \n", " ")
