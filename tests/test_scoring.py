"""Scoring operators without a GPU: refusals (the C checks, compiled by
themselves, and the Python ones), and the oracle's gradients against
differences of its own values."""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest

import scoring_oracle as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, BF16, F16 = 0, 1, 2
P = 1 << 20  # an aligned address that nothing reads


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    """The C argument checks as a library of their own (no CUDA in it)."""
    d = tmp_path_factory.mktemp("args")
    src, lib = str(d / "args.cc"), str(d / "args.so")
    with open(src, "w") as f:
        f.write('#include "ms_scores_args.h"\nextern "C" {\n'
                "const char* logprobs(const void* x, int dt, int64_t B, int64_t V, int64_t ld, double T,"
                " const int32_t* tok, int32_t n, int32_t top, const ms_scores* o) {"
                " return ms::bad_logprobs(x, dt, B, V, ld, T, tok, n, top, o); }\n"
                "const char* backward(const void* x, int dt, int64_t B, int64_t V, int64_t ld, double T,"
                " const int32_t* tok, int32_t n, const double* mx, const double* sm, const float* h,"
                " const float* gl, const float* gh, const void* dx, int64_t dld) {"
                " return ms::bad_logprobs_backward(x, dt, B, V, ld, T, tok, n, mx, sm, h, gl, gh, dx, dld); }\n"
                "const char* distill(const void* x, int dt, int64_t B, int64_t V, int64_t ld, double T,"
                " const int32_t* ids, const float* v, int32_t K, int kind, const float* loss, const void* dx,"
                " int64_t dld) { return ms::bad_distill(x, dt, B, V, ld, T, ids, v, K, kind, loss, dx, dld); }\n}\n")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fPIC", "-shared", "-I",
                    os.path.join(ROOT, "omni.js_b200", "csrc"), src, "-o", lib], check=True)
    L = ctypes.CDLL(lib)
    vp, i, l, d = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_double
    block = [vp, i, l, l, l, d]
    L.logprobs.argtypes = block + [vp, i, i, vp]
    L.backward.argtypes = block + [vp, i, vp, vp, vp, vp, vp, vp, l]
    L.distill.argtypes = block + [vp, vp, i, i, vp, vp, l]
    for f in (L.logprobs, L.backward, L.distill):
        f.restype = ctypes.c_char_p
    return L


GOOD_BLOCK = dict(x=P, dt=F32, B=4, V=100, ld=100, T=1.0)
BAD_BLOCKS = [
    (dict(dt=3), b"dtype"), (dict(dt=-1), b"dtype"), (dict(B=-1), b"B out"), (dict(B=2**31), b"B out"),
    (dict(V=0), b"V out"), (dict(V=65535 * 16384 + 1, ld=2**31), b"V out"), (dict(ld=99), b"ld < V"),
    (dict(ld=2**62), b"too large"), (dict(T=0.0), b"temperature"), (dict(T=-1.0), b"temperature"),
    (dict(T=0.0001), b"temperature"), (dict(T=math.nan), b"temperature"), (dict(T=math.inf), b"temperature"),
    (dict(x=None), b"NULL"), (dict(x=P + 2), b"aligned"), (dict(x=P + 1, dt=BF16), b"aligned"),
]


def _block(**kw):
    return tuple({**GOOD_BLOCK, **kw}[k] for k in ("x", "dt", "B", "V", "ld", "T"))


def test_good_calls_pass_the_checks(checks):
    for kw in (dict(), dict(dt=BF16), dict(dt=F16, x=P + 2), dict(B=0, x=None), dict(B=1, ld=0), dict(V=1, ld=1),
               dict(T=10000.0), dict(B=2**31 - 1, V=1, ld=1)):
        assert checks.logprobs(*_block(**kw), P, 1, 5, P) is None, kw
    assert checks.logprobs(*_block(), None, 0, 256, P) is None
    assert checks.backward(*_block(), P, 256, P, P, None, P, None, 2 * P, 100) is None
    assert checks.backward(*_block(), P, 1, P, P, None, P, None, P, 100) is None  # in place
    assert checks.backward(*_block(), None, 0, P, P, P, None, P, P + 1600, 100) is None  # right behind the logits
    assert checks.distill(*_block(), P, P, 256, 1, P, None, 0) is None
    assert checks.distill(*_block(B=1), P, P, 1, 0, None, P, 0) is None


@pytest.mark.parametrize("kw,why", BAD_BLOCKS)
def test_bad_blocks_are_refused(checks, kw, why):
    b = _block(**kw)
    for got in (checks.logprobs(*b, P, 1, 5, P), checks.backward(*b, P, 1, P, P, None, P, None, 1 << 40, 2**31),
                checks.distill(*b, P, P, 8, 0, P, None, 0)):
        assert got is not None and why in got, (kw, got)


def test_bad_arguments_are_refused(checks):
    lp, bw, ds = checks.logprobs, checks.backward, checks.distill
    b = _block()
    cases = [
        (lp(*b, P, -1, 0, P), b"n_tokens"), (lp(*b, P, 257, 0, P), b"n_tokens"), (lp(*b, P, 1, -1, P), b"top_n"),
        (lp(*b, P, 1, 257, P), b"top_n"), (lp(*b, P, 1, 1, None), b"out is NULL"), (lp(*b, None, 1, 1, P), b"tokens"),
        (bw(*b, None, 1, P, P, None, P, None, 2 * P, 100), b"tokens"),
        (bw(*b, P, 257, P, P, None, P, None, 2 * P, 100), b"n_tokens"),
        (bw(*b, None, 0, P, P, None, P, None, 2 * P, 100), b"without tokens"),
        (bw(*b, P, 1, None, P, None, P, None, 2 * P, 100), b"row_max"),
        (bw(*b, P, 1, P, None, None, P, None, 2 * P, 100), b"row_max"),
        (bw(*b, P, 1, P, P, None, P, P, 2 * P, 100), b"without entropy"),
        (bw(*b, P, 1, P, P, None, P, None, None, 100), b"dlogits is NULL"),
        (bw(*b, P, 1, P, P, None, P, None, 2 * P, 99), b"dld < V"),
        (bw(*b, P, 1, P, P, None, P, None, 2 * P + 2, 100), b"aligned"),
        (bw(*b, P, 1, P, P, None, P, None, P, 101), b"overlaps"),      # the logits with another stride
        (bw(*b, P, 1, P, P, None, P, None, P + 1596, 100), b"overlaps"),
        (bw(*b, P, 1, P, P, None, P, None, P - 4, 100), b"overlaps"),
        (ds(*b, P, P, 0, 0, P, None, 0), b"K must"), (ds(*b, P, P, 257, 0, P, None, 0), b"K must"),
        (ds(*b, P, P, 8, 2, P, None, 0), b"kind"), (ds(*b, None, P, 8, 0, P, None, 0), b"ids/values"),
        (ds(*b, P, None, 8, 0, P, None, 0), b"ids/values"), (ds(*b, P, P, 8, 0, None, None, 0), b"both NULL"),
        (ds(*b, P, P, 8, 0, P, P + 8, 100), b"overlaps"), (ds(*b, P, P, 8, 0, P, 2 * P, 10), b"dld < V"),
    ]
    for i, (got, why) in enumerate(cases):
        assert got is not None and why in got, (i, got)


def test_null_context_is_an_argument_error():
    from minisample import _native as N

    L = N.load()
    s = N.MsScores()
    assert L.ms_logprobs(None, P, F32, 1, 1, 1, 1.0, None, 0, 0, ctypes.byref(s), None) == N.MS_ERR_ARG
    assert L.ms_logprobs_backward(None, P, F32, 1, 1, 1, 1.0, None, 0, P, P, None, None, None, P, 1,
                                  None) == N.MS_ERR_ARG
    assert L.ms_distill(None, P, F32, 1, 1, 1, 1.0, P, P, 1, 0, None, P, None, 0, None) == N.MS_ERR_ARG
    assert L.ms_device(None, None) == N.MS_ERR_ARG


def test_scores_struct_is_six_pointers():
    from minisample._native import MsScores

    assert ctypes.sizeof(MsScores) == 6 * ctypes.sizeof(ctypes.c_void_p)


def test_python_refuses_blocks_that_are_not_on_the_gpu():
    import torch

    from minisample import scoring

    class Stub:
        device_index = 0

    for x in (torch.zeros(2, 3), np.zeros((2, 3), np.float32), torch.zeros(2, 3, dtype=torch.float64)):
        with pytest.raises(ValueError, match="CUDA tensor"):
            scoring._logprobs(Stub(), x, None, 1.0, 0, True, False)


# ---------------------------------------------------------------- the oracle itself
def _row(seed, V=12):
    rng = np.random.default_rng(seed)
    x = rng.normal(0, 2, V)
    x[3] = -np.inf
    return x


def _differences(f, x, h=1e-5):
    g = np.zeros(len(x))
    for i in range(len(x)):
        if np.isfinite(x[i]):
            a, b = x.copy(), x.copy()
            a[i] += h
            b[i] -= h
            g[i] = (f(a) - f(b)) / (2 * h)
    return g


@pytest.mark.parametrize("T", [1.0, 0.7, 2.5])
def test_oracle_score_gradient_against_differences(T):
    x, tok, g, gH = _row(1), [2, 7, 7, -1, 40], [0.5, -1.5, 0.25, 9.0, 9.0], -0.8

    def f(z):
        o, _ = O.score(z, T, tok, 0)
        return float(np.dot(o["logprobs"], g) + gH * o["entropy"])

    dx, _ = O.score_grad(x, T, tok, g, gH, "float32")
    np.testing.assert_allclose(dx, _differences(f, x), atol=1e-8)


@pytest.mark.parametrize("kind", ["logits", "logprobs"])
@pytest.mark.parametrize("T", [1.0, 0.7, 2.5])
def test_oracle_distillation_gradient_against_differences(kind, T):
    x, ids = _row(2), [1, 5, -1, 5, 20, 9]
    v = np.array([0.5, -1.0, 3.0, 0.1, 3.0, -2.0]) if kind == "logits" else np.log([0.3, 0.2, 0.9, 0.1, 0.9, 0.15])

    def f(z):
        return O.distill(z, T, ids, v, kind, 1.0, "float32")[0]

    loss, _, dx, _ = O.distill(x, T, ids, v, kind, 0.6, "float32")
    np.testing.assert_allclose(dx, 0.6 * _differences(f, x), atol=1e-8)
    assert loss > 0


def test_generation_refuses_a_bad_number_of_alternatives():
    """Before the sampler or the model is touched."""
    from minisample.generation import generate_tokens_device, normalize_options

    assert normalize_options({})["logprobs"] is None and normalize_options({"logprobs": 0})["logprobs"] == 0
    for n in (-1, 257, 1.5, True, "5"):
        with pytest.raises(ValueError, match="alternatives"):
            generate_tokens_device(None, [[1]], {"logprobs": n})
