"""What the 8-bit operators refuse, checked without a GPU: the checks run before any kernel is built or launched."""
import pytest
import torch

from tiny_llm_b200 import ops
from tiny_llm_b200.ops import KernelError


@pytest.fixture
def no_device(monkeypatch):
    """The checks of shapes and types on CPU tensors; a call that passes them all ends at the (missing) launch."""
    monkeypatch.setattr(ops, "_fp8_here", lambda *a: None)

    def reached(*_a, **_k):
        raise LookupError("launched")
    monkeypatch.setattr(ops, "_fp8_call", reached)
    monkeypatch.setattr(ops, "status_word", lambda device: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0, raising=False)


def rows(m, k):
    return ops.fp8_rows(m, k, "cpu")


def weight(n, k):
    return ops.fp8_weight(n, k, "cpu")


def test_room_for_rows_and_weights():
    data, scales = rows(3, 130)
    assert data.shape == (3, 130) and data.stride() == (144, 1) and data.dtype == torch.float8_e4m3fn
    assert scales.shape == (3, 2) and scales.dtype == torch.float8_e8m0fnu
    data, scales = weight(257, 128)
    assert data.shape == (257, 128) and data.is_contiguous() and scales.shape == (3, 1) and scales.dtype == torch.float32


def test_tensors_on_the_host_are_refused():
    a, w = rows(2, 128), weight(128, 128)
    for call in (lambda: ops.quantize_fp8(torch.zeros(2, 128), *a), lambda: ops.quantize_weight_fp8(torch.zeros(128, 128), *w),
                 lambda: ops.rms_norm_fp8(torch.zeros(2, 128), torch.zeros(128), 1e-5, *a),
                 lambda: ops.linear_fp8(*a, *w, torch.zeros(2, 128)),
                 lambda: ops.linear_swiglu_fp8(*a, *weight(256, 128), torch.zeros(2, 128, dtype=torch.bfloat16))):
        with pytest.raises(KernelError, match="CUDA device only"):
            call()


def test_calls_that_fit_reach_their_kernel(no_device):
    a, w = rows(2, 200), weight(300, 200)
    wide = torch.zeros(2, 320)
    for call in (lambda: ops.quantize_fp8(torch.zeros(2, 300)[:, 100:], *a), lambda: ops.quantize_fp8(torch.zeros(2, 200, dtype=torch.bfloat16), *a),
                 lambda: ops.quantize_weight_fp8(torch.zeros(300, 200), *w),
                 lambda: ops.rms_norm_fp8(torch.zeros(9, 200), torch.zeros(200), 1e-5, *a, rows=torch.zeros(2, dtype=torch.int32)),
                 lambda: ops.linear_fp8(*a, *w, wide[:, :300]), lambda: ops.linear_fp8(*a, *w, wide[:, 20:], accumulate=True),
                 lambda: ops.linear_fp8(a[0][:1], a[1][:1], *w, torch.zeros(1, 300, dtype=torch.bfloat16)),
                 lambda: ops.linear_swiglu_fp8(*a, *weight(512, 200), *rows(2, 130)),
                 lambda: ops.linear_swiglu_fp8(*a, *weight(512, 200), torch.zeros(2, 256, dtype=torch.bfloat16), act="clamped", limit=1.0)):
        with pytest.raises(LookupError, match="launched"):
            call()


def test_rows_and_weights_that_do_not_fit(no_device):
    a, w = rows(2, 200), weight(300, 200)
    bad_start = torch.zeros(2 * 208 + 8, dtype=torch.uint8)[8:].view(torch.float8_e4m3fn).view(2, 208)[:, :200]
    if bad_start.data_ptr() % 16 == 0:
        bad_start = torch.zeros(2 * 208 + 9, dtype=torch.uint8)[9:].view(torch.float8_e4m3fn).view(2, 208)[:, :200]
    x = torch.zeros(2, 200)
    bad = [
        lambda: ops.quantize_fp8(x.half(), *a),                                                   # a type that no kernel takes
        lambda: ops.quantize_fp8(torch.zeros(200, 2).T, *a),                                      # columns side by side
        lambda: ops.quantize_fp8(torch.zeros(2, 201), *a),
        lambda: ops.quantize_fp8(x, torch.empty(2, 200, dtype=torch.float8_e4m3fn), a[1]),        # rows off 16 bytes
        lambda: ops.quantize_fp8(x, bad_start, a[1]),
        lambda: ops.quantize_fp8(x, a[0].view(torch.uint8), a[1]),
        lambda: ops.quantize_fp8(x, a[0].view(torch.uint8).view(torch.float8_e5m2), a[1]),
        lambda: ops.quantize_fp8(x, a[0], torch.zeros(2, 2)),                                     # scales of another type, shape, order
        lambda: ops.quantize_fp8(x, a[0], rows(2, 300)[1]),
        lambda: ops.quantize_fp8(x, a[0], torch.empty(2, 2, dtype=torch.float8_e8m0fnu).T),
        lambda: ops.quantize_fp8(x, a[0][:1].expand(2, 200), a[1]),                               # one row twice
        lambda: ops.quantize_fp8(x, a[0], a[1][:1].expand(2, 2)),
        lambda: ops.quantize_weight_fp8(torch.zeros(300, 200), w[0], w[1].double()),
        lambda: ops.quantize_weight_fp8(torch.zeros(300, 200), w[0], torch.zeros(3, 3)[:, :2]),
        lambda: ops.quantize_weight_fp8(torch.zeros(200, 300).T, *w),
        lambda: ops.rms_norm_fp8(x.bfloat16(), torch.zeros(200), 1e-5, *a),
        lambda: ops.rms_norm_fp8(torch.zeros(2, 300)[:, :200], torch.zeros(200), 1e-5, *a),
        lambda: ops.rms_norm_fp8(x, torch.zeros(199), 1e-5, *a),
        lambda: ops.rms_norm_fp8(torch.zeros(5, 200), torch.zeros(200), 1e-5, *a),
        lambda: ops.rms_norm_fp8(x, torch.zeros(200), 1e-5, *a, rows=torch.zeros(2, dtype=torch.int64)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(KernelError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_products_that_do_not_fit(no_device):
    a, w, out = rows(2, 200), weight(300, 200), torch.zeros(2, 300)
    half = torch.bfloat16
    bad = [
        lambda: ops.linear_fp8(*rows(2, 208), *w, out),
        lambda: ops.linear_fp8(*a, *w, out[:, :299]),
        lambda: ops.linear_fp8(*a, *w, torch.zeros(3, 300)),
        lambda: ops.linear_fp8(*a, *w, out.half()),
        lambda: ops.linear_fp8(*a, *w, out.to(half), accumulate=True),
        lambda: ops.linear_fp8(*a, *w, torch.zeros(300, 2).T),
        lambda: ops.linear_fp8(*a, *w, out[:1].expand(2, 300)),
        lambda: ops.linear_fp8(a[0], w[1], *w, out),
        lambda: ops.linear_fp8(*a, w[0], w[1][:2], out),
        lambda: ops.linear_fp8(*a, w[0], w[1].T.contiguous().T, out),
        lambda: ops.linear_fp8(a[0].expand(2, 200)[:1].expand(2, 200), a[1], *w, out),
        lambda: ops.linear_fp8(*rows(2, 0), *weight(300, 0), out),
        lambda: ops.linear_swiglu_fp8(*a, *weight(512, 200), torch.zeros(2, 128, dtype=half)),    # rows for another width
        lambda: ops.linear_swiglu_fp8(*a, *weight(400, 200), torch.zeros(2, 200, dtype=half)),    # blocks that are not filled
        lambda: ops.linear_swiglu_fp8(*a, *weight(512, 200), torch.zeros(2, 200)),
        lambda: ops.linear_swiglu_fp8(*a, *weight(512, 200), rows(2, 200)[0]),
        lambda: ops.linear_swiglu_fp8(*a, *weight(512, 200), torch.zeros(2, 200, dtype=half), rows(2, 200)[1]),
        lambda: ops.linear_swiglu_fp8(*a, *weight(512, 200), torch.zeros(2, 200, dtype=half), act="tanh"),
        lambda: ops.linear_swiglu_fp8(*a, *weight(512, 200), torch.zeros(2, 200, dtype=half), act="clamped"),
        lambda: ops.linear_swiglu_fp8(*a, *weight(512, 200), torch.zeros(3, 200, dtype=half)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(KernelError):
            call()
            pytest.fail(f"call {i} was not refused")


# ---------------------------------------------------------------------------------------------- kernels


def test_waits_of_whole_warps_have_one_answer():
    """A wait that gives up may do so in some lanes of a warp and not in others.  Where all lanes wait, the answer goes through a vote before
    anything depends on it; the copying lane, which waits alone, is the only one without."""
    import os
    from tiny_llm_b200.ops import build
    with open(os.path.join(build.CSRC, "linear_fp8.cu")) as f:
        waits = [line.strip() for line in f if "mbar_wait(" in line and not line.lstrip().startswith("//")]
    assert len(waits) == 7
    alone = [w for w in waits if "__all_sync(0xffffffffu," not in w]
    assert len(alone) == 2 and all("mbar_wait(&empty_bar[s]" in w and "ERR_QP_PRODUCER" in w for w in alone)


def test_arguments_have_one_layout():
    """The structs of the entry points are declared once, and the interpreter packs them by what the libraries say."""
    import ctypes
    import os
    import struct
    from tiny_llm_b200.ops import build
    declared = {}
    for name in os.listdir(build.CSRC):
        if name.startswith(("fp8", "linear_fp8")) and not name.endswith(".so"):
            with open(os.path.join(build.CSRC, name)) as f:
                for line in f:
                    if line.startswith("struct ") and "Call {" in line:
                        declared.setdefault(line.split()[1], []).append(name)
    assert declared == {s: ["fp8_calls.h"] for s in ("QuantizeCall", "RmsNormCall", "QuantizeWeightCall", "LinearFp8Call")}
    sizes = {"tllm_quantize_fp8": (10, 72), "tllm_rms_norm_fp8": (11, 80), "tllm_quantize_weight_fp8": (9, 64), "tllm_linear_fp8": (20, 136)}
    for name, (fields, size) in sizes.items():
        letters = getattr(build.load_library(ops._FP8_ENTRIES[name]), name + "_layout")
        letters.restype = ctypes.c_char_p
        assert len(letters()) == fields and struct.calcsize(letters().decode()) == size


def test_sizes_next_to_32_bits_are_refused():
    """Tiles, runs and groups are rounded up in 32 bits: the entry points refuse what that would carry over, before they look at a device."""
    most = 2 ** 31 - 4096
    at = 1 << 20
    entries = {
        "tllm_quantize_fp8": lambda m, k: (at, k, at, 16 * (k // 16 + 1), at, k // 128 + 1, m, k, 0, 0),
        "tllm_rms_norm_fp8": lambda m, k: (at, at, at, 16 * (k // 16 + 1), at, k // 128 + 1, 0, m, k, 1e-5, 0),
        "tllm_quantize_weight_fp8": lambda m, k: (at, k, at, 16 * (k // 16 + 1), at, m, k, 0, 0)}
    for name, args in entries.items():
        for m, k in ((1, most + 1), (1, 2 ** 31 - 1), (most + 1, 16), (2 ** 31 - 1, 128)):
            with pytest.raises(KernelError, match=f"at most {most} rows"):
                ops._fp8_call(name, *args(m, k))
        with pytest.raises(KernelError, match="32 bits"):
            ops._fp8_call(name, *args(2 ** 31, 128))
    for m, n, k, gated in ((most + 1, 8, 8, 0), (8, most + 1, 8, 0), (8, 8, 2 ** 31 - 1, 0), (8, 2 ** 30 + 1, 8, 1), (8, 2 ** 31 - 1, 8, 1)):
        with pytest.raises(KernelError, match=f"at most {most} rows"):
            ops._fp8_call("tllm_linear_fp8", at, 16 * (k // 16 + 1), at, k // 128 + 1, at, 16 * (k // 16 + 1), at, at, n, 0, 0, m, n, k, 0, gated, 0, 0.0, at, 0)


def test_threads_that_load_the_extension_at_once_get_one_module(monkeypatch, tmp_path):
    """In a fresh build folder, with a compiler that takes its time, so that they do meet."""
    import shutil
    import threading
    from tiny_llm_b200.ops import build
    source = tmp_path / "csrc"
    source.mkdir()
    (source / "two_threads.cpp").write_text("""#include <Python.h>
        static PyModuleDef module = {PyModuleDef_HEAD_INIT, "two_threads", nullptr, -1, nullptr, nullptr, nullptr, nullptr, nullptr};
        PyMODINIT_FUNC PyInit_two_threads(void) { return PyModule_Create(&module); }""")
    slow = tmp_path / "slow_compiler"
    slow.write_text(f"#!/bin/sh\nsleep 1\n{shutil.which('g++')} \"$@\"\nstatus=$?\nsleep 1\nexit $status\n")
    slow.chmod(0o755)
    monkeypatch.setattr(build, "CSRC", str(source))
    monkeypatch.setenv("TLLM_BUILD_DIR", str(tmp_path / "build"))
    monkeypatch.setenv("CXX", str(slow))
    modules, errors = [], []

    def load():
        try:
            modules.append(build.load_extension("two_threads"))
        except Exception as e:
            errors.append(e)
    threads = [threading.Thread(target=load) for _ in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    assert len(modules) == 3 and all(m is modules[0] for m in modules) and modules[0].__name__ == "two_threads"


# ---------------------------------------------------------------------------------------------- models


def test_the_engine_refuses_what_has_no_8_bit_form():
    from conftest import TINY_A
    from tiny_llm_b200.config import LlamaConfig, config_from_dict
    from tiny_llm_b200.engine.loading import parse_weights
    from tiny_llm_b200.parts import DecoderModel
    import dunelix_util

    assert parse_weights(None, torch.float32) is False and parse_weights("fp8", torch.bfloat16) is True
    for weights, dtype in (("fp8", torch.float32), ("int4", torch.bfloat16)):
        with pytest.raises(ValueError):
            parse_weights(weights, dtype)
    model = DecoderModel(LlamaConfig.from_dict(TINY_A).model_spec())
    with pytest.raises(RuntimeError, match="no weights"):
        model.to_fp8()
    model.load({n: torch.zeros([s or 1 for s in w.shape]) for n, w in model.weight_specs().items()})
    with pytest.raises(ValueError, match="bfloat16 engine"):
        model.to_fp8()
    other = DecoderModel(config_from_dict(next(v for v in vars(dunelix_util).values() if isinstance(v, dict) and v.get("architecture") == "Dunelix")).model_spec())
    other.loaded = True
    with pytest.raises(ValueError, match="without an 8-bit form"):
        other.to_fp8()


def test_the_command_line_takes_the_form_of_the_weights():
    from tiny_llm_b200.__main__ import parse_flags
    assert parse_flags(["--weights=fp8"])["weights"] == "fp8" and parse_flags([])["weights"] == ""


@pytest.fixture
def small_model(monkeypatch):
    """A loaded bfloat16 decoder on the host, whose matrices turn to 8 bits in plain arithmetic."""
    import fp8_util as fu
    from conftest import TINY_A
    from tiny_llm_b200.config import LlamaConfig
    from tiny_llm_b200.parts import DecoderModel

    def to_fp8(w):
        q, s = fu.quantize_weight(w)
        return q.float().to(torch.float8_e4m3fn), s.float()
    monkeypatch.setattr(ops, "weight_to_fp8", to_fp8)
    model = DecoderModel(LlamaConfig.from_dict(TINY_A).model_spec())
    weights = {n: torch.ones([s or 1 for s in w.shape], dtype=torch.bfloat16) for n, w in model.weight_specs().items()}
    model.load(weights)
    return model, weights


def test_a_model_that_a_runner_uses_is_not_turned(small_model):
    from tiny_llm_b200.engine.loading import make_runner
    model, _ = small_model
    before = [(b.mixer.w_qkv, b.ffn.w_down) for b in model.blocks]
    make_runner(model, "bfloat16", "cpu", max_tokens=64)
    with pytest.raises(RuntimeError, match="a runner was built"):
        model.to_fp8()
    assert all(b.mixer.w_qkv is x and b.ffn.w_down is y and not b.mixer.fp8 and not b.ffn.fp8 for b, (x, y) in zip(model.blocks, before))


def test_a_model_in_8_bits_stays_so(small_model):
    from tiny_llm_b200.engine.loading import make_runner
    model, _ = small_model
    model.to_fp8()
    held = [b.mixer.w_qkv for b in model.blocks]
    make_runner(model, "bfloat16", "cpu", max_tokens=64)
    model.to_fp8()
    assert all(b.mixer.w_qkv is x and b.mixer.fp8 and b.ffn.fp8 for b, x in zip(model.blocks, held))


def test_a_model_in_8_bits_loads_again(small_model):
    """New weights are bfloat16 matrices again, whole layers of them, until the model is turned again."""
    model, weights = small_model
    model.to_fp8()
    assert all(isinstance(x, tuple) for b in model.blocks for x in (b.mixer.w_qkv, b.mixer.w_o, b.ffn.w_gate_up, b.ffn.w_down))
    model.load(weights)
    assert all(isinstance(x, torch.Tensor) for b in model.blocks for x in (b.mixer.w_qkv, b.mixer.w_o, b.ffn.w_gate_up, b.ffn.w_down))
    assert not any(b.mixer.fp8 or b.ffn.fp8 for b in model.blocks)
    model.to_fp8()
    assert all(isinstance(b.ffn.w_down, tuple) and isinstance(b.mixer.w_o, tuple) for b in model.blocks)


def test_turning_a_model_goes_on_where_it_broke_off(small_model, monkeypatch):
    model, _ = small_model
    turn, calls = ops.weight_to_fp8, []

    def breaks(w):
        calls.append(w)
        if len(calls) == 4:      # the first layer's down matrix
            raise MemoryError
        return turn(w)
    monkeypatch.setattr(ops, "weight_to_fp8", breaks)
    with pytest.raises(MemoryError):
        model.to_fp8()
    first = model.blocks[0]
    assert first.mixer.fp8 and not first.ffn.fp8 and isinstance(first.ffn.w_gate_up, torch.Tensor) and isinstance(first.ffn.w_down, torch.Tensor)
    model.to_fp8()
    assert all(b.mixer.fp8 and b.ffn.fp8 and isinstance(b.ffn.w_gate_up, tuple) and isinstance(b.ffn.w_down, tuple) for b in model.blocks)
