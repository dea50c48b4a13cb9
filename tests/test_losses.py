"""The softmax losses' argument checks (no GPU): every refusal of the C
entries comes before anything is enqueued, so host addresses stand in for
device memory here."""
from __future__ import annotations

import ctypes as C
import os
import re
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

import distlr_amd as dlr  # noqa: E402
import distlr_amd.losses as L  # noqa: E402
from conftest import ROOT  # noqa: E402

BUF = (C.c_char * 65536)()
BASE = (C.addressof(BUF) + 255) // 256 * 256
A, B, D, E, F = (BASE + 8192 * i for i in range(5))


HEADER = os.path.join(ROOT, "include", "distlr_losses.h")


def test_header_library_and_binding_agree():
    with open(HEADER) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(dlr_[a-z0-9_]+)\s*\(", text)))
    out = subprocess.run(["nm", "-D", "--defined-only", L.LIB_PATH], check=True, capture_output=True, text=True).stdout
    exported = {line.split()[-1] for line in out.splitlines() if line.strip()}
    assert sorted(L.SYMBOLS) == declared and set(declared) <= exported
    with open(L.LIB_PATH, "rb") as f:
        assert b"amdgcn-amd-amdhsa--gfx950" in f.read()


@pytest.mark.parametrize("language", ["c", "c++"])
def test_header_stands_alone(language):
    subprocess.run(["g++", "-fsyntax-only", "-Wall", "-Werror", "-x", language, "-I", os.path.join(ROOT, "include"), "-"],
                   input=b'#include "distlr_losses.h"\n', check=True)


@pytest.mark.parametrize("order", ["torch, distlr_amd.losses", "distlr_amd, torch, distlr_amd.losses",
                                   "distlr_amd.losses"])
def test_the_library_takes_torchs_runtime_in_any_order_of_imports(order):
    prog = (f"import sys; sys.path.insert(0, {os.path.join(ROOT, 'dist-lr_amd')!r})\n"
            f"import {order}\nimport torch, distlr_amd.losses as L, os\n"
            "own = os.path.join(os.path.dirname(torch.__file__), 'lib', 'libamdhip64.so')\n"
            "print(not os.path.exists(own) or os.path.samefile(L.lib.dlr_losses_runtime().decode(), own))")
    out = subprocess.run([sys.executable, "-c", prog], check=True, capture_output=True, text=True).stdout
    assert out.strip() == "True"


def code(rc):
    assert rc < 0
    return rc, L.lib.dlr_losses_last_error().decode()


def logits(**kw):
    x = dict(data=A, target=B, rows=4, vocab=8, row_stride=8, dtype=L.DTYPE_F32, target_bits=64, temperature=1.0)
    x.update(kw)
    return L._Logits(**x)


BAD_LOGITS = [
    (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 30) + 1), "vocab"),
    (dict(row_stride=7), "row_stride"), (dict(row_stride=-8), "row_stride"), (dict(row_stride=1 << 62), "row_stride"),
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(data=None), "NULL"), (dict(data=A + 2), "aligned"),
    (dict(target=None), "target"), (dict(target=B + 4), "target"), (dict(target_bits=16), "target_bits"),
    (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"),
    (dict(temperature=float("nan")), "temperature"), (dict(temperature=float("inf")), "temperature"),
    (dict(temperature=1e-9), "temperature"),
]


@pytest.mark.parametrize("kw,word", BAD_LOGITS, ids=lambda v: str(v)[:40])
def test_bad_logits_are_refused_by_every_call(kw, word):
    x, p = logits(**kw), L._Policy(D, None, D, None, 0.2, 0.2, 0.0)
    for rc in (L.lib.dlr_token_logprob(0, None, C.byref(x), None, 0, D, E),
               L.lib.dlr_token_logprob_grad(0, None, C.byref(x), D, D, E, 8),
               L.lib.dlr_policy_loss(0, None, C.byref(x), C.byref(p), None, 0, E, E, E, E, None, 0)):
        rc, msg = code(rc)
        assert rc == dlr.E_ARG and word in msg


def test_null_descriptors_and_outputs():
    x, p = logits(), L._Policy(D, None, D, None, 0.2, 0.2, 0.0)
    calls = [
        lambda: L.lib.dlr_token_logprob(0, None, None, None, 0, D, E),
        lambda: L.lib.dlr_token_logprob(0, None, C.byref(x), None, 0, None, E),
        lambda: L.lib.dlr_token_logprob(0, None, C.byref(x), None, 0, D, None),
        lambda: L.lib.dlr_token_logprob(0, None, C.byref(x), None, 0, D + 2, E),
        lambda: L.lib.dlr_token_logprob_grad(0, None, C.byref(x), None, D, E, 8),
        lambda: L.lib.dlr_token_logprob_grad(0, None, C.byref(x), D, None, E, 8),
        lambda: L.lib.dlr_token_logprob_grad(0, None, C.byref(x), D, D, None, 8),
        lambda: L.lib.dlr_policy_loss(0, None, C.byref(x), None, None, 0, E, E, E, E, None, 0),
        lambda: L.lib.dlr_policy_loss(0, None, C.byref(x), C.byref(p), None, 0, None, E, E, E, None, 0),
        lambda: L.lib.dlr_policy_loss(0, None, C.byref(x), C.byref(p), None, 0, E, E, E, None, None, 0),
        lambda: L.lib.dlr_preference_loss(0, None, None, E, E, E, None),
        lambda: L.lib.dlr_head_logprob(0, None, None, D, 1 << 20, E, E),
    ]
    for call in calls:
        assert code(call())[0] == dlr.E_ARG


@pytest.mark.parametrize("grad,stride,word", [
    (D, 7, "grad_row_stride"), (D, -8, "grad_row_stride"), (D + 2, 8, "aligned"), (A + 4, 8, "overlap"),
    (A, 9, "overlap"), (A + 4 * 31, 8, "overlap"), (A - 4, 8, "overlap")])
def test_gradients_that_do_not_fit(grad, stride, word):
    x, p = logits(), L._Policy(E, None, E, None, 0.2, 0.2, 0.0)
    for rc in (L.lib.dlr_token_logprob_grad(0, None, C.byref(x), E, E, grad, stride),
               L.lib.dlr_policy_loss(0, None, C.byref(x), C.byref(p), None, 0, F, F, F, F, grad, stride)):
        rc, msg = code(rc)
        assert rc == dlr.E_ARG and word in msg


def test_gradient_over_logits_whose_rows_share_memory():
    x = logits(row_stride=0)
    rc, msg = code(L.lib.dlr_token_logprob_grad(0, None, C.byref(x), E, E, A, 0))
    assert rc == dlr.E_ARG


@pytest.mark.parametrize("kw,word", [
    (dict(clip_low=-0.1), "clip_low"), (dict(clip_low=1.1), "clip_low"), (dict(clip_low=float("nan")), "clip_low"),
    (dict(clip_high=-0.1), "clip_high"), (dict(clip_high=float("inf")), "clip_high"), (dict(kl_coef=-1.0), "kl_coef"),
    (dict(kl_coef=float("nan")), "kl_coef"), (dict(kl_coef=0.1, ref_logprob=None), "ref_logprob"),
    (dict(old_logprob=None), "old_logprob"), (dict(advantage=None), "advantage"), (dict(weight=D + 1), "aligned")])
def test_bad_policy(kw, word):
    v = dict(old_logprob=D, ref_logprob=D, advantage=D, weight=None, clip_low=0.2, clip_high=0.2, kl_coef=0.1)
    v.update(kw)
    x, p = logits(), L._Policy(**v)
    rc, msg = code(L.lib.dlr_policy_loss(0, None, C.byref(x), C.byref(p), None, 0, E, E, E, E, None, 0))
    assert rc == dlr.E_ARG and word in msg


@pytest.mark.parametrize("kw,word", [
    (dict(pairs=-1), "pairs"), (dict(pairs=1 << 30), "pairs"), (dict(tokens=-1), "tokens"), (dict(beta=0.0), "beta"),
    (dict(beta=float("inf")), "beta"), (dict(label_smoothing=-0.1), "label_smoothing"),
    (dict(label_smoothing=1.5), "label_smoothing"), (dict(margin=float("nan")), "margin"), (dict(average=2), "average"),
    (dict(offsets=None), "offsets"), (dict(offsets=B + 4), "offsets"), (dict(logprob=None), "logprob"),
    (dict(ref_logprob=A + 2), "aligned")])
def test_bad_preference(kw, word):
    v = dict(logprob=A, ref_logprob=A, mask=None, offsets=B, weight=None, pairs=2, tokens=10, beta=0.1,
             label_smoothing=0.0, margin=0.0, average=0, reserved=0)
    v.update(kw)
    p = L._Preference(**v)
    rc, msg = code(L.lib.dlr_preference_loss(0, None, C.byref(p), D, D, D, E))
    assert rc == dlr.E_ARG and word in msg


def test_preference_gradient_over_an_input():
    p = L._Preference(A, None, None, B, None, 2, 10, 0.1, 0.0, 0.0, 0, 0)
    rc, msg = code(L.lib.dlr_preference_loss(0, None, C.byref(p), D, D, D, A + 8))
    assert rc == dlr.E_ARG and "overlap" in msg


@pytest.mark.parametrize("kw,word", [
    (dict(rows=-1), "rows"), (dict(vocab=0), "vocab"), (dict(dim=0), "dim"), (dict(dim=(1 << 20) + 1), "dim"),
    (dict(rows=1 << 30, vocab=1 << 20), "rows"),
    (dict(dtype=L.DTYPE_F32), "dtype"), (dict(hidden=None), "NULL"), (dict(head=A + 1), "aligned"),
    (dict(hidden_stride=63), "hidden_stride"), (dict(head_stride=63), "head_stride"), (dict(head_stride=0), "head_stride"),
    (dict(target=None), "target"), (dict(temperature=0.0), "temperature")])
def test_bad_head(kw, word):
    v = dict(hidden=A, head=A, target=B, rows=4, vocab=100, dim=64, hidden_stride=64, head_stride=64,
             dtype=L.DTYPE_BF16, target_bits=64, temperature=1.0)
    v.update(kw)
    h = L._Head(**v)
    rc, msg = code(L.lib.dlr_head_logprob(0, None, C.byref(h), D, 1 << 30, E, E))
    assert rc == dlr.E_ARG and word in msg


def test_head_workspace():
    need = L.lib.dlr_head_logprob_workspace(4, 100, 64)
    assert need > 0
    assert code(L.lib.dlr_head_logprob_workspace(4, 0, 64))[0] == dlr.E_ARG
    h = L._Head(A, A, B, 4, 100, 64, 64, 64, L.DTYPE_BF16, 64, 1.0)
    for ws, size in ((None, need), (D, need - 1), (D + 4, need)):
        rc, msg = code(L.lib.dlr_head_logprob(0, None, C.byref(h), ws, size, E, E))
        assert rc == dlr.E_ARG and "workspace" in msg


def test_logits_workspace():
    size = L.lib.dlr_logits_workspace
    assert size(1, 32000, L.DTYPE_BF16) == 0 and size(129, 1 << 20, L.DTYPE_F32) == 0 and size(0, 1 << 20, 0) == 0
    for rows, vocab, dtype in ((0, 0, 0), (-1, 9, 0), (4, (1 << 30) + 1, 0), (4, 100, 3)):
        assert code(size(rows, vocab, dtype))[0] == dlr.E_ARG
    need = size(4, 200000, L.DTYPE_BF16)
    assert need > 0
    assert all(size(r, v, d) == 0 for r in (1, 128) for v in (1, 32767) for d in range(3))  # what the binding skips
    x = logits(rows=4, vocab=200000, row_stride=200000, dtype=L.DTYPE_BF16)
    p = L._Policy(D, None, D, None, 0.2, 0.2, 0.0)
    for ws, n in ((None, need), (E, need - 1), (E + 4, need)):
        for rc in (L.lib.dlr_token_logprob(0, None, C.byref(x), ws, n, D, E),
                   L.lib.dlr_policy_loss(0, None, C.byref(x), C.byref(p), ws, n, D, D, D, D, None, 0)):
            rc, msg = code(rc)
            assert rc == dlr.E_ARG and "workspace" in msg


def test_a_device_that_is_not_there():
    x, p = logits(), L._Policy(D, None, D, None, 0.2, 0.2, 0.0)
    q = L._Preference(A, None, None, B, None, 2, 10, 0.1, 0.0, 0.0, 0, 0)
    h = L._Head(A, A, B, 4, 100, 64, 64, 64, L.DTYPE_BF16, 64, 1.0)
    for rc in (L.lib.dlr_token_logprob(99, None, C.byref(x), None, 0, D, E),
               L.lib.dlr_token_logprob_grad(99, None, C.byref(x), D, D, E, 8),
               L.lib.dlr_policy_loss(99, None, C.byref(x), C.byref(p), None, 0, E, E, E, E, None, 0),
               L.lib.dlr_preference_loss(99, None, C.byref(q), D, D, D, E),
               L.lib.dlr_head_logprob(99, None, C.byref(h), D, 1 << 20, E, E)):
        assert code(rc)[0] == -4  # DLR_E_HIP


def test_no_rows_is_a_valid_call():
    x, p = logits(rows=0, data=None, target=None), L._Policy(None, None, None, None, 0.2, 0.2, 0.0)
    assert L.lib.dlr_token_logprob(0, None, C.byref(x), None, 0, None, None) == 0
    assert L.lib.dlr_token_logprob_grad(0, None, C.byref(x), None, None, None, 0) == 0
    assert L.lib.dlr_policy_loss(0, None, C.byref(x), C.byref(p), None, 0, None, None, None, None, None, 0) == 0
    q = L._Preference(None, None, None, None, None, 0, 0, 0.1, 0.0, 0.0, 0, 0)
    assert L.lib.dlr_preference_loss(0, None, C.byref(q), None, None, None, None) == 0
    h = L._Head(None, None, None, 0, 100, 64, 64, 64, L.DTYPE_BF16, 64, 1.0)
    assert L.lib.dlr_head_logprob(0, None, C.byref(h), None, 0, None, None) == 0


@pytest.mark.parametrize("struct,name", [(L._Logits, "dlr_logits"), (L._Policy, "dlr_policy"),
                                         (L._Preference, "dlr_preference"), (L._Head, "dlr_head")])
def test_structs_match_the_header(struct, name):
    with open(HEADER) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
    ctype = {"const void *": C.c_void_p, "const float *": C.c_void_p, "const uint8_t *": C.c_void_p,
             "const int64_t *": C.c_void_p, "int64_t": C.c_int64, "int32_t": C.c_int32, "double": C.c_double}
    fields = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        kind, names = re.match(r"((?:const )?\w+ ?\*?)\s*(.*)", decl, re.S).groups()
        fields += [(n.strip(), ctype[kind.strip()]) for n in names.split(",")]
    assert fields == [(n, t) for n, t in struct._fields_]


def test_tensors_off_the_gpu_are_refused():
    z, y, v = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64), torch.zeros(3)
    for call in (lambda: L.token_logprob(z, y), lambda: L.token_logprob_grad(z, y, v, v),
                 lambda: L.policy_loss(z, y, v, v), lambda: L.preference_loss(v, v, y, beta=0.1),
                 lambda: L.head_logprob(z, z, y), lambda: L.token_logprob([1.0], y)):
        with pytest.raises(dlr.DLRError) as e:
            call()
        assert e.value.code == dlr.E_ARG


def test_calls_beyond_one_launch():
    # more pairs or classes than a launch has threads for are refused, more rows go by several launches
    p = L._Preference(A, None, None, B, None, 1 << 22, 10, 0.1, 0.0, 0.0, 0, 0)
    rc, msg = code(L.lib.dlr_preference_loss(0, None, C.byref(p), D, D, D, E))
    assert rc == dlr.E_ARG and "pairs" in msg
    size = L.lib.dlr_head_logprob_workspace
    assert code(size(1, (1 << 28) + 1, 64))[0] == dlr.E_ARG and size(1, 1 << 28, 64) > 0
    h = L._Head(A, A, B, 1, (1 << 28) + 1, 64, 64, 64, L.DTYPE_BF16, 64, 1.0)
    rc, msg = code(L.lib.dlr_head_logprob(0, None, C.byref(h), D, 1 << 40, E, E))
    assert rc == dlr.E_ARG and "vocab" in msg
    # scratch memory is a slice's, whatever the call's rows (a tile's 8 bytes a row, at most one for 64 classes)
    for vocab in (7, 4096, 131072, 1 << 24):
        most = min(1 << 21, (1 << 35) // vocab)
        for rows in (most, most + 1, 2 * most + 1, 5 * most, min((1 << 31) - 1, (1 << 44) // vocab)):
            need = size(rows, vocab, 512)
            assert need <= most * 8 * (vocab // 64 + 3) + 512
            slices = -(-rows // most)
            each = -(-rows // slices)
            assert need >= size(each, vocab, 512) and need >= size(rows - (rows - 1) // each * each, vocab, 512)
