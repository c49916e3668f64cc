"""Arguments of the layer, norm and row functions that are refused, before anything reaches a device."""
import math

import pytest
import torch


def test_fused_linear_refuses():
    import ash

    x, w, b = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(5)
    bad = [
        dict(x=x, weight=torch.zeros(5, 7)), dict(x=x, weight=torch.zeros(8)), dict(x=torch.zeros(()), weight=w),
        dict(x=torch.zeros(3, 0), weight=torch.zeros(5, 0)), dict(x=x, weight=torch.zeros(0, 8)),
        dict(x=x.double(), weight=w.double()), dict(x=x, weight=w.half()), dict(x=x.int(), weight=w.int()),
        dict(x=x, weight=w, bias=torch.zeros(4)), dict(x=x, weight=w, bias=torch.zeros(1, 5)), dict(x=x, weight=w, bias=b.half()),
        dict(x=x, weight=w, residual=torch.zeros(5)), dict(x=x, weight=w, residual=torch.zeros(3, 5).bfloat16()),
        dict(x=x, weight=w, activation="tanh"), dict(x=x, weight=w, activation="sin", omega=math.inf),
        dict(x=x, weight=w, dtype=torch.float16), dict(x=x, weight=None if False else "w"),
        dict(x=[1.0], weight=w),
    ]
    for kw in bad:
        with pytest.raises((ValueError, AttributeError)):
            ash.fused_linear(**kw)


def test_quantised_operands_refuse():
    import ash

    rows = lambda n, k, dtype=torch.float8_e4m3fn, s=torch.float32: ash.QuantizedRows(torch.zeros(n, k).to(dtype),
                                                                                  torch.ones(n, dtype=s))
    x, w = rows(3, 8), rows(5, 8)
    bad = [
        (x, torch.zeros(5, 8), {}), (torch.zeros(3, 8), w, {}), (x, rows(5, 9), {}), (rows(3, 8, torch.int8), w, {}),
        (x, rows(5, 8, torch.uint8), {}), (x, rows(5, 8, s=torch.float64), {}), (x, w, {"dtype": torch.float64}),
        (x, w, {"bias": torch.zeros(5)}), (x, w, {"residual": torch.zeros(3, 5, dtype=torch.float16)}),
        (ash.QuantizedRows(x.codes, torch.ones(4)), w, {}), (ash.QuantizedRows(x.codes, torch.ones(3, 1)), w, {}),
        (ash.QuantizedRows([1], x.scales), w, {}),
    ]
    for a, b, kw in bad:
        with pytest.raises(ValueError):
            ash.fused_linear(a, b, **kw)
    bias = torch.zeros(5, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(RuntimeError, match="gradient"):
        ash.fused_linear(x, w, bias)


def test_rms_norm_refuses():
    import ash

    x, w = torch.zeros(3, 8), torch.ones(8)
    for kw in [dict(x=x, weight=torch.ones(7)), dict(x=x, weight=w.half()), dict(x=x.double(), weight=w.double()),
               dict(x=torch.zeros(3, 0), weight=torch.ones(0)), dict(x=torch.zeros(()), weight=w), dict(x=x, weight=w, eps=-1.0),
               dict(x=x, weight=w, eps=math.nan), dict(x=x, weight=w, residual=torch.zeros(1, 8)),
               dict(x=x, weight=w, residual=torch.zeros(3, 8).half())]:
        with pytest.raises(ValueError):
            ash.rms_norm(**kw)
    with pytest.raises(RuntimeError, match="gradient"):
        ash.rms_norm(x.requires_grad_(True), w, quantize=True)


def test_rows_refuse():
    import ash

    x = torch.zeros(3, 8)
    for bad in (lambda: ash.quantize_rows(x, "int4"), lambda: ash.quantize_rows(x.double()), lambda: ash.quantize_rows(x.int()),
                lambda: ash.quantize_rows(torch.zeros(())), lambda: ash.quantize_rows(torch.zeros(3, 0)),
                lambda: ash.dequantize_rows(ash.QuantizedRows(x.to(torch.int8), torch.ones(2))),
                lambda: ash.dequantize_rows(ash.QuantizedRows(x.to(torch.int8), torch.ones(3)), dtype=torch.float64),
                lambda: ash.dequantize_rows(ash.QuantizedRows(x.to(torch.int8), torch.ones(3)), torch.zeros(2, dtype=torch.int32)),
                lambda: ash.dequantize_rows(ash.QuantizedRows(x.to(torch.int8)[None], torch.ones(1, 3)),
                                            torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(ValueError):
            bad()


def test_map_formats_refuse():
    import ash
    from ash.hashmap import _value_formats

    assert _value_formats(None, 4) == {} and _value_formats("int8", [1, 2]) == {"default_0": "int8", "default_1": "int8"}
    assert _value_formats([None, "e4m3"], [1, 2]) == {"default_1": "e4m3"}
    assert _value_formats({"b": "e4m3"}, {"a": 1, "b": 2}) == {"b": "e4m3"}
    for formats, dims in [("int4", 4), (["int8"], 4), (["int8"], [1, 2]), ({"c": "int8"}, {"a": 1}), (["int8", 3], [1, 2]),
                          ("int8", {"a": 1, "a_scale": 1}), ("int8", 0)]:
        with pytest.raises(ValueError):
            _value_formats(formats, dims)
    if not torch.cuda.is_available():       # a stand-in of the native module has no rows in 8 bits
        with pytest.raises(RuntimeError):
            ash.HashMap(3, 4, 10, "cpu", value_formats="int8")


def test_modules_refuse():
    import ash
    from ash.mlp import Linear

    for bad in (lambda: Linear(0, 3), lambda: Linear(3, 0), lambda: Linear(3, 3, activation="tanh"), lambda: ash.MLP(3, 8, 1, 0),
                lambda: ash.SirenNet(3, 8, 1, 0), lambda: ash.ResidualMLP(3, 8, 1, 0), lambda: ash.ResidualMLP(3, 8, 1, 1, 0)):
        with pytest.raises(ValueError):
            bad()


def test_library_refuses_cpu_tensors_and_bad_arguments():
    """The shim and the C entry points themselves: nothing is launched."""
    import ctypes
    import importlib.util
    import os

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    spec = importlib.util.spec_from_file_location("_shim_of_layers", os.path.join(root, "torch-ash_b200", "__ash.py"))
    shim = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(shim)
    x, w = torch.zeros(3, 8), torch.zeros(5, 8)
    for call in (lambda: shim.linear_forward(x, w, None, "none", None, 1.0, False),
                 lambda: shim.rms_norm_forward(x, torch.ones(8), None, 1e-6, False, False),
                 lambda: shim.quantize_rows(x, torch.int8), lambda: shim.read_rows(x.to(torch.int8), torch.ones(3), None, torch.float32)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    lib, p = shim._lib, ctypes.c_void_p(4096)
    f = lambda *a: lib.ashb_linear_forward(*a)
    good = [0, p, 8, None, p, 8, None, None, None, 0, 3, 8, 5, 0, 1.0, 0, p, None, None, 0, None]
    for at, value in [(0, 1), (0, 9), (2, 7), (5, 7), (10, -1), (11, 0), (12, 0), (13, 5), (15, 3), (16, None), (1, None), (17, p)]:
        args = list(good)
        args[at] = value
        if at == 17:
            args[10] = 100       # a slope without an activation
        assert f(*args) == 1, (at, value, lib.ashb_last_error_string())
    args = list(good)
    args[0] = 8                  # e4m3 without scales
    assert f(*args) == 1
    args = list(good)
    args[2], args[10] = 9, 100   # rows that are no whole words, and no workspace for their copy
    assert f(*args) == 1 and lib.ashb_linear_forward_workspace(0, p, 9, p, 8, 100, 8, 5) == 3328      # 100 rows of 32 bytes
    assert lib.ashb_linear_forward_workspace(0, p, 8, p, 8, 100, 8, 5) == 0 == lib.ashb_linear_forward_workspace(0, p, 9, p, 8, 4, 8, 5)
    assert lib.ashb_linear_backward(0, p, None, 1, p, 8, p, 8, 3, 8, 5, p, p, p, None, 0, None) == 1
    assert lib.ashb_linear_backward(0, p, p, 1, p, 8, p, 8, 3000, 8, 5, p, p, p, p, 8, None) == 1       # small workspace
    assert lib.ashb_rms_norm_forward(0, p, 4, None, 0, p, 3, 8, 1e-6, p, None, None, None, None, None) == 1
    assert lib.ashb_rms_norm_forward(0, p, 8, None, 0, p, 3, 8, 1e-6, p, p, p, None, None, None) == 1
    assert lib.ashb_rms_norm_forward(0, p, 8, p, 8, p, 3, 8, 1e-6, p, None, None, None, None, None) == 1
    assert lib.ashb_rms_norm_backward(0, p, None, p, p, p, 3, 8, p, p, p, 0, None) == 1
    t = shim._RowTable(4096, 4096, 4096, 8, 3, 0)
    assert lib.ashb_quantize_rows(4, ctypes.byref(t), None) == 1
    t = shim._RowTable(4096, 4096, None, 8, 1, 0)
    assert lib.ashb_quantize_rows(4, ctypes.byref(t), None) == 1
    t = shim._RowTable(4096, 4096, 4096, 8, 1, 1)
    assert lib.ashb_read_rows(4, None, 4, ctypes.byref(t), None) == 1
    t = shim._RowTable(4096, 4096, 4096, 8, 1, 0)
    assert lib.ashb_read_rows(5, None, 4, ctypes.byref(t), None) == 1
    assert lib.ashb_map_insert_rows(None, p, 3, 0, None, p, None) == 1 and lib.ashb_map_find_rows(None, p, 3, p, p, 0, None, None) == 1


def test_waits_that_ran_out_raise(monkeypatch):
    """check_waits of a stand-in that counts, and the library's knob."""
    import ash

    asked = []
    for count in (0, 3):
        monkeypatch.setattr(ash.mlp, "backend", type("Counts", (), {"layer_timeouts": staticmethod(lambda d: asked.append(d) or count)}))
        for device in (1, "cuda:1", torch.device("cuda", 1)):
            if count:
                with pytest.raises(RuntimeError, match="3 thread blocks on cuda:1"):
                    ash.mlp.check_waits(device)
            else:
                assert ash.mlp.check_waits(device) is None
    assert asked == [torch.device("cuda", 1)] * 6
