"""Refusals of the scoring calls and options that need no GPU."""
import asyncio

import pytest


class _NoModel:
    """A model that must not be touched."""

    def __getattr__(self, name):
        raise AssertionError(f"{name} of the model was used")


def test_loops_without_log_probabilities_refuse_the_option():
    """Only generate_tokens_device returns them; the others say so instead of leaving them out."""
    from minisample import generation as G

    for n in (0, 5):
        opts = {"maxNewTokens": 2, "logprobs": n}
        for call in (lambda: G.generate_tokens(_NoModel(), [1], opts),
                     lambda: G.generate_tokens_batch(_NoModel(), [[1], [2]], opts),
                     lambda: asyncio.run(G.generate_async(_NoModel(), [1], opts))):
            with pytest.raises(ValueError, match="generate_tokens_device"):
                call()
    with pytest.raises(AssertionError):  # None is no such request
        G.generate_tokens(_NoModel(), [1], {"maxNewTokens": 2, "logprobs": None})


# ---------------------------------------------------------------- the C entry points' checks
def _pointer_checks(d):
    """The argument checks that look at pointers, compiled by themselves."""
    import ctypes
    import os
    import subprocess

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src, lib = str(d / "args.cc"), str(d / "args.so")
    with open(src, "w") as f:
        f.write('#include "ms_scores_args.h"\nextern "C" {\n'
                "const char* scores(const void* tok, float* lp, float* h, int32_t* ids, float* top, double* mx, double* sm) {"
                " ms_scores o = {lp, h, ids, top, mx, sm}; const void* x = (const void*)64;"
                " const char* e = ms::bad_logprobs(x, MS_F32, 2, 8, 8, 1.0, (const int32_t*)tok, 1, 1, &o);"
                " return e ? e : ms::bad_scores(o); }\n"
                "const char* backward(const int32_t* tok, const double* mx, const double* sm, const float* h,"
                " const float* gl, const float* gh) { return ms::bad_logprobs_backward((const void*)64, MS_F32, 2, 8, 8,"
                " 1.0, tok, 1, mx, sm, h, gl, gh, (const void*)4096, 8); }\n"
                "const char* distill(const int32_t* ids, const float* v, const float* loss, const float* w) {"
                " return ms::bad_distill((const void*)64, MS_F32, 2, 8, 8, 1.0, ids, v, 3, 0, loss, nullptr, 0, w); }\n}\n")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fPIC", "-shared", "-I",
                    os.path.join(root, "omni.js_b200", "csrc"), src, "-o", lib], check=True)
    L = ctypes.CDLL(lib)
    for f, n in ((L.scores, 7), (L.backward, 6), (L.distill, 4)):
        f.restype, f.argtypes = ctypes.c_char_p, [ctypes.c_void_p] * n
    return L


def test_pointers_that_are_not_aligned_are_refused(tmp_path):
    """An access through one would be a fault of the GPU; NULL where it is allowed stays allowed."""
    L = _pointer_checks(tmp_path)
    P = 1 << 20
    cases = [  # call, its good arguments, the alignment of each, which may be NULL
        (L.scores, 7, [4, 4, 4, 4, 4, 8, 8], [1, 2, 3, 4, 5, 6]),
        (L.backward, 6, [4, 8, 8, 4, 4, 4], [3, 4, 5]),
        (L.distill, 4, [4, 4, 4, 4], [3]),
    ]
    for call, n, sizes, optional in cases:
        assert call(*[P] * n) is None
        for i in range(n):
            for off in range(1, sizes[i]):
                a = [P] * n
                a[i] += off
                got = call(*a)
                assert got is not None and b"aligned" in got, (call.__name__, i, off, got)
            if i in optional and not (call is L.backward and i == 3):  # g_entropy needs entropy
                a = [P] * n
                a[i] = None
                assert call(*a) is None, (call.__name__, i)
