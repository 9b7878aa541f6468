"""The MLP-block operators without a GPU: what their descriptors refuse before
any CUDA call, their buffer sizes, and what the torch-facing shim refuses."""
import contextlib
import ctypes
import sys

import pytest
import torch

import sp24

P = 0x10000   # a non-null, 16-byte aligned "pointer"; refused calls never read it


def _fill(d, base, kw):
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    return ctypes.byref(d)


ROWS = dict(dtype=1, qdtype=sp24.I8, rows=4, cols=64, x=P, q=P, scale=P)


@pytest.mark.parametrize("entry,kw,code", [
    ("sp24_quantize_rows", dict(dtype=2), 8),                    # 16-bit rows only
    ("sp24_quantize_rows", dict(dtype=sp24.I8), 8),
    ("sp24_quantize_rows", dict(qdtype=5), 8),                   # e5m2 codes are not offered
    ("sp24_quantize_rows", dict(qdtype=1), 8),
    ("sp24_quantize_rows", dict(cols=0), 1),
    ("sp24_quantize_rows", dict(rows=-1), 1),
    ("sp24_quantize_rows", dict(ldx=63), 1),
    ("sp24_quantize_rows", dict(ldq=8), 1),
    ("sp24_quantize_rows", dict(x=None), 8),
    ("sp24_quantize_rows", dict(q=None), 8),
    ("sp24_quantize_rows", dict(scale=None), 8),
    ("sp24_quantize_rows", dict(weight=P), 8),                   # another operator's fields
    ("sp24_quantize_rows", dict(up=P), 8),
    ("sp24_quantize_rows", dict(residual=P), 8),
    ("sp24_swiglu_quant", dict(), 8),                            # no up
    ("sp24_swiglu_quant", dict(up=P, ld_up=32), 1),
    ("sp24_swiglu_quant", dict(up=P, residual_out=P), 8),
    ("sp24_rmsnorm_quant", dict(), 8),                           # no weight
    ("sp24_rmsnorm_quant", dict(weight=P, eps=-1.0), 8),
    ("sp24_rmsnorm_quant", dict(weight=P, eps=float("nan")), 8),
    ("sp24_rmsnorm_quant", dict(weight=P, up=P), 8),
    ("sp24_rmsnorm_quant", dict(weight=P, residual_out=P), 8),   # a sum of nothing
    ("sp24_rmsnorm_quant", dict(weight=P, residual=P, ld_residual=8), 1),
    ("sp24_quantize_rows", dict(rows=0, x=None, q=None, scale=None), 0),
])
def test_rows_refusals(entry, kw, code):
    lib = sp24.load()
    assert getattr(lib, entry)(_fill(sp24.RowQuantDesc(), ROWS, kw), None) == code
    assert getattr(lib, entry)(None, None) == 8


SCALED = dict(dtype=sp24.I8, cdtype=1, m=128, n=16, k=128, a_c=P, meta=P, x=P, c=P)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=1), 8), (dict(dtype=5), 8), (dict(dtype=7), 8),
    (dict(cdtype=2), 8), (dict(cdtype=sp24.I8), 8),
    (dict(m=0), 1), (dict(n=-1), 1), (dict(k=0), 1), (dict(k=96), 1),
    (dict(k=131136), 1),                      # int8 sums could leave 32 bits
    (dict(lda_c=32), 1), (dict(ldx=64), 1), (dict(ldc=64), 1),
    (dict(a_c=None), 8), (dict(meta=None), 8), (dict(x=None), 8), (dict(c=None), 8),
    (dict(a_c=P + 8), 2), (dict(x=P + 4), 2), (dict(meta=P + 2), 2),
    (dict(lda_c=72), 2), (dict(ldx=136), 2),
    (dict(n=0, x=None, c=None), 0),
])
def test_scaled_refusals(kw, code):
    lib = sp24.load()
    assert lib.sp24_gemm_scaled(_fill(sp24.ScaledDesc(), SCALED, kw), None) == code
    assert lib.sp24_gemm_scaled(None, None) == 8


FFN = dict(dtype=1, t=4, h=64, f=96, act=1, x=P, w_gate=P, w_up=P)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), 8), (dict(dtype=7), 8), (dict(act=3), 8), (dict(act=-1), 8),
    (dict(t=-1), 1), (dict(h=0), 1), (dict(f=0), 1),
    (dict(ldx=63), 1), (dict(ld_gate=56), 1), (dict(ld_up=8), 1),
    (dict(x=None), 8), (dict(w_gate=None), 8), (dict(w_up=None), 8),
    (dict(x=P + 2), 2), (dict(w_up=P + 8), 2), (dict(ldx=68), 2), (dict(h=63), 2),
    (dict(saved=P, saved_bytes=4 * 2 * 128 * 4 - 1), 9),
    (dict(t=0, x=None), 0),
])
def test_ffn_forward_refusals(kw, code):
    lib = sp24.load()
    assert lib.sp24_ffn_forward(_fill(sp24.FfnDesc(), FFN, kw), P, 0, None) == code
    assert lib.sp24_ffn_forward(None, P, 0, None) == 8
    assert lib.sp24_ffn_forward(_fill(sp24.FfnDesc(), FFN, {}), None, 0, None) == 8
    assert lib.sp24_ffn_forward(_fill(sp24.FfnDesc(), FFN, {}), P, 95, None) == 1


@pytest.mark.parametrize("kw,gkw,code", [
    ({}, dict(dw_up=None), 8),                # one weight gradient without the other
    ({}, dict(d_out=None), 8),
    (dict(saved=None), {}, 8),
    (dict(saved_bytes=100), {}, 9),
    ({}, dict(workspace=None), 9),
    ({}, dict(workspace_bytes=100), 9),
    ({}, dict(workspace=P + 4), 2),
    ({}, dict(ld_d_out=95), 1),
    ({}, dict(ld_dx=63), 1),
    ({}, dict(ld_dgate=63), 1),
    (dict(act=3), {}, 8),
])
def test_ffn_backward_refusals(kw, gkw, code):
    lib = sp24.load()
    need = lib.sp24_ffn_workspace_bytes(4, 64, 96)
    base = dict(FFN, saved=P, saved_bytes=lib.sp24_ffn_saved_bytes(4, 96))
    grads = dict(d_out=P, dx=P, dw_gate=P, dw_up=P, workspace=P, workspace_bytes=need)
    d = _fill(sp24.FfnDesc(), base, kw)
    assert lib.sp24_ffn_backward(d, _fill(sp24.FfnGrads(), grads, gkw), None) == code
    assert lib.sp24_ffn_backward(d, None, None) == 8


def test_ffn_buffer_sizes():
    lib = sp24.load()
    assert lib.sp24_ffn_saved_bytes(3, 10) == 3 * 2 * 64 * 4     # rows of 64 values
    assert lib.sp24_ffn_workspace_bytes(3, 8, 10) == 3 * 2 * 64 * 2   # one slice: dg and du alone
    # 2 x 20 stages, slices of at least eight: five planes of 3 x 64 sums
    assert lib.sp24_ffn_workspace_bytes(3, 8, 1280) == 3 * 2 * 1280 * 2 + 5 * 3 * 64 * 4
    assert lib.sp24_ffn_saved_bytes(0, 10) == lib.sp24_ffn_workspace_bytes(5, 8, 0) == 0
    assert lib.sp24_ffn_saved_bytes(70000, 14336) == 70000 * 2 * 14336 * 4   # past 32 bits


def test_plain_gemm_still_refuses_the_new_types():
    lib = sp24.load()
    d = sp24.GemmDesc()
    d.m = d.n = d.k = 128
    d.a_c = d.meta = d.b = d.c_f32 = P
    d.meta_format = sp24.META_TC
    for dtype in (sp24.I8, sp24.F32):
        d.dtype = dtype
        assert lib.sp24_gemm(ctypes.byref(d), None) == 8
        assert lib.sp24_prune_2of4(dtype, P, 8, 8, 0, P, 0, None) == 8
    assert lib.sp24_repack_meta(sp24.F32, P, 64, 64, P, None) == 8
    assert lib.sp24_repack_meta(sp24.I8, P, 64, 32, P, None) == 1    # k % 64 as for fp8


def test_fused_gemm_still_refuses_the_new_activation():
    lib = sp24.load()
    d = sp24.GemmDesc()
    d.m = d.n = d.k = 128
    d.a_c = d.meta = d.b = d.c_f32 = P
    d.meta_format = sp24.META_TC
    e = sp24.Epilogue()
    e.act = sp24.ACT_GELU_TANH
    assert lib.sp24_gemm_fused(ctypes.byref(d), ctypes.byref(e), None) == 8


def test_shim_refusals():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        sp24.quantize_rows(x, qdtype=sp24.E5M2)
    with pytest.raises(ValueError):
        sp24.quantize_rows(x.float())
    with pytest.raises(ValueError):
        sp24.swiglu_quant(x, x.half())
    with pytest.raises(ValueError):
        sp24.gemm_scaled(x, x, x)
    with pytest.raises(ValueError):
        sp24.ffn_gated(x, x.half(), x)
    with pytest.raises(ValueError):
        sp24.ffn_gated_backward(x.half(), x, x, x, x)


def test_packed_descriptors_match_the_structures():
    """The shim's packed descriptors are the ctypes structures byte for byte."""
    for pack, cls in ((sp24._PACK_ROWS, sp24.RowQuantDesc), (sp24._PACK_SCALED, sp24.ScaledDesc),
                      (sp24._PACK_FFN, sp24.FfnDesc), (sp24._PACK_GRADS, sp24.FfnGrads)):
        values = [float(i) + 0.5 if t is ctypes.c_float else i + 1 for i, (_, t) in enumerate(cls._fields_)]
        want = cls(*values)
        got = pack(*values)
        assert len(got) <= ctypes.sizeof(cls)
        back = cls.from_buffer_copy(got.ljust(ctypes.sizeof(cls), b"\0"))
        assert [getattr(back, n) for n, _ in cls._fields_] == [getattr(want, n) for n, _ in cls._fields_]


@pytest.mark.parametrize("step,aligned", [(64, True), (72, False), (65, False)])
def test_copied_weights_lose_the_static_hint(monkeypatch, step, aligned):
    """Weights that the shim copies on the stream are in-flight work of the
    call: it is launched without the hint, and the caller's hint stays set."""
    real, seen = sp24.load(), []

    class Library:
        def __getattr__(self, name):
            return getattr(real, name)

        def sp24_gemm_scaled(self, *args):
            seen.append(real.sp24_get_launch_hints())
            return 0

        sp24_ffn_forward = sp24_gemm_scaled

    monkeypatch.setattr(sp24, "_lib", Library())
    a_c = torch.zeros(128, step, dtype=torch.int8)[:, :64]
    x8 = torch.zeros(4, 128, dtype=torch.int8)
    image = torch.zeros(sp24.meta_tc_bytes(128, 128), dtype=torch.uint8)
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    w = torch.zeros(96, 64, dtype=torch.bfloat16)
    odd = torch.zeros(96, 64 if aligned else 65, dtype=torch.bfloat16)[:, :64]
    for hints in (sp24.HINT_NONE, sp24.HINT_STATIC_WEIGHTS):
        sp24.set_launch_hints(hints)
        try:
            sp24._gemm_scaled(0, a_c, image, x8, None, None, None, None)
            sp24._ffn_forward(0, x, w, odd, sp24.ACT_SILU, False)
            sp24._ffn_forward(0, x, odd, w, sp24.ACT_SILU, False)
            assert sp24.get_launch_hints() == hints
        finally:
            sp24.set_launch_hints(sp24.HINT_NONE)
        # tokens may be copied: they are loaded after the wait in any case
        sp24._ffn_forward(0, torch.zeros(4, 65, dtype=torch.bfloat16)[:, :64], w, w, sp24.ACT_SILU, False)
        want = hints if aligned else sp24.HINT_NONE
        assert seen == [want, want, want, sp24.HINT_NONE]
        seen.clear()


def test_type_tables_are_published_whole(monkeypatch):
    """What another thread finds at every line of the first call that builds the
    tables: nothing, or all of them."""
    whole = set(sp24._code_tables())
    monkeypatch.setattr(sp24, "_codes", {})
    seen = []

    def trace(frame, event, arg):
        if frame.f_code is sp24._code_tables.__code__:
            seen.append(set(sp24._codes))
            return trace

    before = sys.gettrace()
    sys.settrace(trace)
    try:
        sp24._code_tables()
    finally:
        sys.settrace(before)
    assert len(seen) > 2 and all(s in (set(), whole) for s in seen) and set(sp24._codes) == whole


def test_first_calls_from_several_threads_in_a_fresh_process():
    """Threads whose very first calls meet: each gets its own refusal (tensors
    without a GPU), past the type tables."""
    import os
    import subprocess
    code = """
import sys, threading
sys.path.insert(0, sys.argv[1])
sys.setswitchinterval(1e-6)
import torch
import sp24
x = torch.zeros(4, 64, dtype=torch.bfloat16)
x8, image = torch.zeros(4, 128, dtype=torch.int8), torch.zeros(4096, dtype=torch.uint8)
gate, failed = threading.Barrier(8), []
def first(i):
    gate.wait()
    for call in (lambda: sp24._ffn_args(x, x, x, sp24.ACT_SILU),
                 lambda: sp24._gemm_scaled(0, x8.float(), image, x8, None, None, None, None),
                 lambda: sp24._rows_quant(0, "sp24_quantize_rows", x.float(), sp24.I8, None, None, None, 0.0)):
        try:
            call()
        except ValueError:
            pass
        except Exception as e:
            failed.append(repr(e))
for _ in range(50):
    sp24._codes = {}
    threads = [threading.Thread(target=first, args=(i,)) for i in range(8)]
    [t.start() for t in threads]
    [t.join() for t in threads]
assert not failed, failed
"""
    subprocess.run([sys.executable, "-c", code, os.path.dirname(sp24.__file__)], check=True, timeout=300)


@pytest.mark.parametrize("current", [0, 1])
def test_streams_of_another_device_are_refused(monkeypatch, current):
    """A named stream has to be one of the tensors' device: entering it would
    make its own device current, and the launch would go there."""
    class Stream:
        device_index = 1

    launched = []
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current, raising=False)
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "stream", lambda stream: contextlib.nullcontext())
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    with pytest.raises(ValueError, match="stream of cuda:1"):
        sp24._on(0, Stream(), launched.append)
    assert not launched
    sp24._on(1, Stream(), launched.append)
    assert launched == [0]


@pytest.mark.parametrize("form", ["plain", "strided", "expanded"])
def test_strided_images_and_saved_buffers_are_read_as_they_are_indexed(monkeypatch, form):
    """The metadata image and the saved buffer go to the library as plain bytes:
    strided ones are copied first, and none is read past its own storage."""
    real, seen = sp24.load(), []

    class Library:
        def __getattr__(self, name):
            return getattr(real, name)

        def sp24_gemm_scaled(self, d, stream):
            desc = sp24.ScaledDesc.from_buffer_copy(d.ljust(ctypes.sizeof(sp24.ScaledDesc), b"\0"))
            seen.append((ctypes.string_at(desc.meta, 4096), real.sp24_get_launch_hints()))
            return 0

        def sp24_ffn_backward(self, d, grads, stream):
            desc = sp24.FfnDesc.from_buffer_copy(d.ljust(ctypes.sizeof(sp24.FfnDesc), b"\0"))
            seen.append((ctypes.string_at(desc.saved, desc.saved_bytes), None))
            return 0

    def strided(v):
        if form == "strided":
            wide = torch.zeros(2 * v.numel(), dtype=v.dtype)
            wide[::2] = v
            return wide[::2]
        return v[:1].expand(v.numel()) if form == "expanded" else v

    monkeypatch.setattr(sp24, "_lib", Library())
    image = strided(torch.randint(0, 256, (4096,), dtype=torch.uint8))
    sp24.set_launch_hints(sp24.HINT_STATIC_WEIGHTS)
    try:
        sp24._gemm_scaled(0, torch.zeros(128, 64, dtype=torch.int8), image, torch.zeros(4, 128, dtype=torch.int8),
                          None, None, None, None)
    finally:
        sp24.set_launch_hints(sp24.HINT_NONE)
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(96, 64, dtype=torch.bfloat16)
    saved = strided(torch.randint(0, 256, (real.sp24_ffn_saved_bytes(4, 96),), dtype=torch.uint8))
    sp24._ffn_backward(0, torch.zeros(4, 96, dtype=torch.bfloat16), x, w, w, saved, sp24.ACT_SILU, True, True)
    # an image that was copied is in-flight work: the launch goes without the hint
    hints = sp24.HINT_STATIC_WEIGHTS if form == "plain" else sp24.HINT_NONE
    assert seen == [(bytes(image.tolist()), hints), (bytes(saved.tolist()), None)]


def test_type_and_shape_refusals_by_their_own_message():
    """The checks that follow the one for a GPU, reached without it."""
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    x8, image = torch.zeros(4, 128, dtype=torch.int8), torch.zeros(4096, dtype=torch.uint8)
    a_c = torch.zeros(128, 64, dtype=torch.int8)

    def rows(x, qdtype=sp24.I8, up=None, weight=None, residual=None):
        return sp24._rows_quant(0, "sp24_rows", x, qdtype, up, weight, residual, 0.0)

    for message, call in (
            ("qdtype 5", lambda: rows(x, sp24.E5M2)),
            ("float16 or bfloat16 rows, not torch.float32", lambda: rows(x.float())),
            ("torch.float16 beside torch.bfloat16", lambda: rows(x, up=x.half())),
            ("x: a 2-D tensor", lambda: rows(x[0])),
            ("up: shape", lambda: rows(x, up=x[:, :32])),
            ("weight: shape", lambda: rows(x, weight=x[0, :32])),
            ("residual: shape", lambda: rows(x, residual=x[:2])),
            ("tokens and", lambda: sp24._gemm_scaled(0, a_c.float(), image, x8, None, None, None, None)),
            ("out_dtype", lambda: sp24._gemm_scaled(0, a_c, image, x8, None, None, None, torch.int8)),
            ("meta_tc: 4080 bytes", lambda: sp24._gemm_scaled(0, a_c, image[16:], x8, None, None, None, None)),
            ("scale_w: 128", lambda: sp24._gemm_scaled(0, a_c, image, x8, torch.ones(4), None, None, None)),
            ("scale_x: 4", lambda: sp24._gemm_scaled(0, a_c, image, x8, None, torch.ones(4).double(), None, None)),
            ("one of float16 and", lambda: sp24._ffn_args(x, x.half(), x, sp24.ACT_SILU)),
            ("w_up: shape", lambda: sp24._ffn_args(x, x, x[:2], sp24.ACT_SILU)),
            ("torch.float16 beside", lambda: sp24._ffn_backward(0, x.half(), x, x, x, image, 1, True, True)),
            ("d_out: shape", lambda: sp24._ffn_backward(0, x, x, x, x, image, 1, True, True))):
        with pytest.raises(ValueError, match=message):
            call()
    with pytest.raises(ValueError, match="CUDA tensors are wanted"):
        sp24.quantize_rows(x)
