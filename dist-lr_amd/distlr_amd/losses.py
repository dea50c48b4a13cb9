"""Softmax losses on torch tensors (include/distlr_losses.h).

Log-probabilities of given classes and their gradient, the paired logistic
(preference) loss, the clipped policy loss, and log-probabilities straight
from hidden states and the output layer's weights.

The many-class counterparts of the engine's margin, residual and log-loss
(lr.cc:35-40, 47-63).  Like the engine they return gradients, they do not
record an autograd graph: pass one on with ``logits.backward(grad)``.

Every tensor is on one GPU.  The work runs on torch's current stream of that
GPU and may be captured into a graph; results and scratch memory come from
torch's allocator.  As with torch's own operators, a tensor made on another
stream has to be waited for by the caller.  Arguments that do not fit raise
``DLRError`` with code ``E_ARG`` before anything is enqueued.
"""
from __future__ import annotations

import ctypes as C
import os
from typing import NamedTuple, Optional, Tuple

import torch

from . import E_ARG, PKG, DLRError, _two_runtimes

LIB_PATH = os.path.join(PKG, "lib", "libdistlr_losses.so")
LIB_PATH = os.environ.get("DLR_LOSSES_LIB", LIB_PATH)  # as DLR_LIB: a variant build of the same library

if not os.path.exists(LIB_PATH):
    raise ImportError(f"{LIB_PATH} not built: run `make -C dist-lr_amd` (or __graft_entry__.build())")

lib = C.CDLL(LIB_PATH)  # after torch: it takes the runtime torch has loaded

P, i64 = C.c_void_p, C.c_int64
SYMBOLS = {
    "dlr_losses_last_error": (C.c_char_p,),
    "dlr_losses_runtime": (C.c_char_p,),
    "dlr_logits_workspace": (i64, i64, i64, C.c_int),
    "dlr_token_logprob": (C.c_int, C.c_int, P, P, P, i64, P, P),
    "dlr_token_logprob_grad": (C.c_int, C.c_int, P, P, P, P, P, i64),
    "dlr_policy_loss": (C.c_int, C.c_int, P, P, P, P, i64, P, P, P, P, P, i64),
    "dlr_preference_loss": (C.c_int, C.c_int, P, P, P, P, P, P),
    "dlr_head_logprob_workspace": (i64, i64, i64, i64),
    "dlr_head_logprob": (C.c_int, C.c_int, P, P, P, i64, P, P),
}
for _name, (_res, *_args) in SYMBOLS.items():
    getattr(lib, _name).restype, getattr(lib, _name).argtypes = _res, _args

_runtime = os.path.join(os.path.dirname(torch.__file__), "lib", "libamdhip64.so")  # where torch brings its own
if os.path.exists(_runtime) and not os.path.samefile(lib.dlr_losses_runtime().decode(), _runtime):
    raise ImportError(f"{LIB_PATH} is bound to {lib.dlr_losses_runtime().decode()}, not to torch's HIP runtime")

DTYPE_F32, DTYPE_BF16, DTYPE_F16 = 0, 1, 2
_DTYPES = {torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16, torch.float16: DTYPE_F16}
_TARGET_BITS = {torch.int32: 32, torch.int64: 64}


def _check(rc: int) -> int:
    if rc < 0:
        raise DLRError(rc, lib.dlr_losses_last_error().decode(errors="replace"))
    return rc


class _Logits(C.Structure):
    _fields_ = [("data", C.c_void_p), ("target", C.c_void_p), ("rows", C.c_int64), ("vocab", C.c_int64),
                ("row_stride", C.c_int64), ("dtype", C.c_int32), ("target_bits", C.c_int32),
                ("temperature", C.c_double)]


class _Policy(C.Structure):
    _fields_ = [("old_logprob", C.c_void_p), ("ref_logprob", C.c_void_p), ("advantage", C.c_void_p),
                ("weight", C.c_void_p), ("clip_low", C.c_double), ("clip_high", C.c_double), ("kl_coef", C.c_double)]


class _Preference(C.Structure):
    _fields_ = [("logprob", C.c_void_p), ("ref_logprob", C.c_void_p), ("mask", C.c_void_p), ("offsets", C.c_void_p),
                ("weight", C.c_void_p), ("pairs", C.c_int64), ("tokens", C.c_int64), ("beta", C.c_double),
                ("label_smoothing", C.c_double), ("margin", C.c_double), ("average", C.c_int32),
                ("reserved", C.c_int32)]


class _Head(C.Structure):
    _fields_ = [("hidden", C.c_void_p), ("head", C.c_void_p), ("target", C.c_void_p), ("rows", C.c_int64),
                ("vocab", C.c_int64), ("dim", C.c_int64), ("hidden_stride", C.c_int64), ("head_stride", C.c_int64),
                ("dtype", C.c_int32), ("target_bits", C.c_int32), ("temperature", C.c_double)]


class PolicyLoss(NamedTuple):
    """Per row; grad has the logits' shape and type (None if not asked for)."""
    loss: torch.Tensor
    logprob: torch.Tensor
    kl: torch.Tensor
    clipped: torch.Tensor
    grad: Optional[torch.Tensor]


class PreferenceLoss(NamedTuple):
    """Per pair; grad is per token (None if not asked for)."""
    loss: torch.Tensor
    chosen_reward: torch.Tensor
    rejected_reward: torch.Tensor
    grad: Optional[torch.Tensor]


def _refuse(why: str):
    raise DLRError(E_ARG, why)


def _gpu(name: str, t) -> int:
    """The index of the tensor's GPU."""
    if not isinstance(t, torch.Tensor):
        _refuse(f"{name} must be a torch tensor")
    if not t.is_cuda:
        _refuse(f"{name} must be on a GPU (it is on {t.device})" + ("" if torch.cuda.is_available() else _two_runtimes()))
    return t.get_device()


def _matrix(name: str, t: torch.Tensor, gpu: int) -> None:
    if _gpu(name, t) != gpu:
        _refuse(f"{name} is on GPU {t.get_device()}, not on GPU {gpu}")
    _rows_of(name, t)


def _rows_of(name: str, t: torch.Tensor) -> None:
    if t.dim() != 2:
        _refuse(f"{name} must have 2 dimensions (it has {t.dim()})")
    if t.stride(1) != 1 and t.shape[1] > 1:
        _refuse(f"{name} must be contiguous within a row")


def _vector(name: str, t, gpu: int, dtypes, length: int) -> torch.Tensor:
    """A 1-D tensor of one of `dtypes`; a strided one is copied."""
    if (isinstance(t, torch.Tensor) and t.is_cuda and t.get_device() == gpu and t.dtype in dtypes
            and t.shape == (length,)):
        return t if t.is_contiguous() else t.contiguous()
    if _gpu(name, t) != gpu:
        _refuse(f"{name} is on GPU {t.get_device()}, not on GPU {gpu}")
    if t.dtype not in dtypes:
        _refuse(f"{name} must be {' or '.join(str(d) for d in dtypes)} (it is {t.dtype})")
    _refuse(f"{name} must have shape ({length},) (it has {tuple(t.shape)})")


_F32 = (torch.float32,)
_INTS = (torch.int64, torch.int32)
_BOOL = (torch.bool,)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _logits(logits: torch.Tensor, target: torch.Tensor, temperature: float):
    gpu = _gpu("logits", logits)
    _rows_of("logits", logits)
    if logits.dtype not in _DTYPES:
        _refuse(f"logits must be float32, bfloat16 or float16 (they are {logits.dtype})")
    rows, vocab = logits.shape
    target = _vector("target", target, gpu, _INTS, rows)
    return gpu, target, _Logits(logits.data_ptr(), target.data_ptr(), rows, vocab, logits.stride(0),
                                _DTYPES[logits.dtype], _TARGET_BITS[target.dtype], temperature)


def _grad_like(logits: torch.Tensor, out: Optional[torch.Tensor], gpu: int) -> torch.Tensor:
    if out is None:
        return torch.empty_like(logits, memory_format=torch.contiguous_format)  # half of torch.empty's 2.3 us
    _matrix("out", out, gpu)
    if out.dtype != logits.dtype or out.shape != logits.shape:
        _refuse("out must have the logits' type and shape")
    return out


def _written(out: Optional[torch.Tensor]) -> None:
    """Autograd sees that a tensor of the caller's, which it may have saved, was written."""
    if out is not None and not out.is_inference():
        torch.autograd.graph.increment_version(out)


def _rows(out: torch.Tensor):
    """Vectors side by side in one allocation, and its address."""
    return out.unbind(0), out.data_ptr()


def _scratch(x: _Logits, like: torch.Tensor):
    """dlr_logits_workspace's bytes and memory (kept until the launch; the
    allocator keeps it for the stream).  Most calls need none."""
    if x.rows > 128 or x.vocab < 32768:
        return 0, None
    need = _check(lib.dlr_logits_workspace(x.rows, x.vocab, x.dtype))
    return need, torch.empty(need, dtype=torch.uint8, device=like.device) if need else None


# The current stream of a GPU as an address: torch.cuda.current_stream(gpu).
# cuda_stream without the Stream object, 2 us of a 10 us call.
_stream = torch._C._cuda_getCurrentRawStream


def token_logprob(logits: torch.Tensor, target: torch.Tensor, *,
                  temperature: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(logprob, lse), float32 per row: logprob = logits[t, target[t]] /
    temperature - lse, lse = log sum exp(logits[t] / temperature).  A
    negative target marks a row that takes no part: 0, not read
    (dlr_token_logprob)."""
    gpu, target, x = _logits(logits, target, temperature)
    out, at = _rows(torch.empty((2, x.rows), dtype=torch.float32, device=logits.device))
    need, scratch = _scratch(x, logits)
    _check(lib.dlr_token_logprob(gpu, _stream(gpu), C.byref(x), _ptr(scratch), need, at, at + 4 * x.rows))
    return out


def token_logprob_grad(logits: torch.Tensor, target: torch.Tensor, lse: torch.Tensor, grad: torch.Tensor, *,
                       temperature: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient with respect to the logits of sum(grad * logprob), in the
    logits' type; lse is token_logprob's, or that of more classes than these.
    Rows with a negative target or grad 0 are 0.  out may be the logits
    themselves (dlr_token_logprob_grad)."""
    gpu, target, x = _logits(logits, target, temperature)
    lse = _vector("lse", lse, gpu, _F32, x.rows)
    grad = _vector("grad", grad, gpu, _F32, x.rows)
    dz = _grad_like(logits, out, gpu)
    _check(lib.dlr_token_logprob_grad(gpu, _stream(gpu), C.byref(x), lse.data_ptr(), grad.data_ptr(),
                                      dz.data_ptr(), dz.stride(0)))
    _written(out)
    return dz


def policy_loss(logits: torch.Tensor, target: torch.Tensor, old_logprob: torch.Tensor, advantage: torch.Tensor, *,
                ref_logprob: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0, temperature: float = 1.0,
                grad: bool = True, out: Optional[torch.Tensor] = None) -> PolicyLoss:
    """The clipped policy loss with a KL term, per row, and the gradient of
    sum(weight * loss) with respect to the logits, in one pass
    (dlr_policy_loss).

    loss = -min(ratio A, clip(ratio, 1 - clip_low, 1 + clip_high) A) +
    kl_coef kl, ratio = exp(logprob - old_logprob), kl = exp(ref - logprob) -
    (ref - logprob) - 1 (0 without ref_logprob).  weight defaults to 1: give
    each row its share of a mean.  Rows with a negative target or weight 0
    take no part.  clipped: where the clip holds the surrogate.  out: the
    gradient's tensor, which may be the logits themselves."""
    gpu, target, x = _logits(logits, target, temperature)
    rows = x.rows
    old_logprob = _vector("old_logprob", old_logprob, gpu, _F32, rows)
    advantage = _vector("advantage", advantage, gpu, _F32, rows)
    if ref_logprob is not None:
        ref_logprob = _vector("ref_logprob", ref_logprob, gpu, _F32, rows)
    if weight is not None:
        weight = _vector("weight", weight, gpu, _F32, rows)
    if out is not None and not grad:
        _refuse("out is the gradient's tensor: grad must be True")
    dz = _grad_like(logits, out, gpu) if grad else None
    p = _Policy(old_logprob.data_ptr(), _ptr(ref_logprob), advantage.data_ptr(), _ptr(weight), clip_low, clip_high,
                kl_coef)
    (loss, logprob, kl), at = _rows(old_logprob.new_empty((3, rows)))  # float32: 0.3 us less than torch.empty
    clipped = torch.empty(rows, dtype=torch.bool, device=logits.device)
    need, scratch = _scratch(x, logits)
    _check(lib.dlr_policy_loss(gpu, _stream(gpu), C.byref(x), C.byref(p), _ptr(scratch), need, at, at + 4 * rows,
                               at + 8 * rows, clipped.data_ptr(), _ptr(dz), 0 if dz is None else dz.stride(0)))
    _written(out)
    return PolicyLoss(loss, logprob, kl, clipped, dz)


def preference_loss(logprob: torch.Tensor, ref_logprob: Optional[torch.Tensor], offsets: torch.Tensor, *, beta: float,
                    label_smoothing: float = 0.0, margin: float = 0.0, mask: Optional[torch.Tensor] = None,
                    weight: Optional[torch.Tensor] = None, average: bool = False,
                    grad: bool = True) -> PreferenceLoss:
    """The paired logistic loss over packed sequences of token
    log-probabilities, per pair, and the gradient of sum(weight * loss) with
    respect to logprob (dlr_preference_loss).

    offsets (int64, 2 P + 1 ascending): sequence i is tokens [offsets[i],
    offsets[i + 1]); pair p compares sequence p (preferred) with P + p.
    reward = beta * sum(logprob - ref_logprob) over the tokens with mask
    (average: per counted token); loss = -(1 - label_smoothing) log sigma(u) -
    label_smoothing log sigma(-u), u = chosen_reward - rejected_reward -
    margin.  weight (P) defaults to 1."""
    gpu = _gpu("logprob", logprob)
    if logprob.dim() != 1:
        _refuse(f"logprob must have 1 dimension (it has {logprob.dim()})")
    tokens = logprob.shape[0]
    logprob = _vector("logprob", logprob, gpu, _F32, tokens)
    if ref_logprob is not None:
        ref_logprob = _vector("ref_logprob", ref_logprob, gpu, _F32, tokens)
    _gpu("offsets", offsets)
    if offsets.dim() != 1 or offsets.shape[0] % 2 != 1:
        _refuse("offsets must have 2 P + 1 entries")
    pairs = offsets.shape[0] // 2
    offsets = _vector("offsets", offsets, gpu, (torch.int64,), 2 * pairs + 1)
    if mask is not None:
        mask = _vector("mask", mask, gpu, _BOOL, tokens)
    if weight is not None:
        weight = _vector("weight", weight, gpu, _F32, pairs)
    p = _Preference(logprob.data_ptr(), _ptr(ref_logprob), _ptr(mask), offsets.data_ptr(), _ptr(weight), pairs, tokens,
                    beta, label_smoothing, margin, 1 if average else 0, 0)
    (loss, chosen, rejected), at = _rows(logprob.new_empty((3, pairs)))
    dl = torch.empty_like(logprob) if grad else None
    _check(lib.dlr_preference_loss(gpu, _stream(gpu), C.byref(p), at, at + 4 * pairs, at + 8 * pairs, _ptr(dl)))
    return PreferenceLoss(loss, chosen, rejected, dl)


def head_logprob(hidden: torch.Tensor, head: torch.Tensor, target: torch.Tensor, *,
                 temperature: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """token_logprob of the logits hidden (rows x dim) . head^T (vocab x dim),
    which are never written out: scoring by a model that is not trained.
    bfloat16 or float16, sums in 32 bits (dlr_head_logprob)."""
    gpu = _gpu("hidden", hidden)
    _rows_of("hidden", hidden)
    _matrix("head", head, gpu)
    if hidden.dtype not in (torch.bfloat16, torch.float16) or head.dtype != hidden.dtype:
        _refuse(f"hidden and head must both be bfloat16 or float16 (they are {hidden.dtype} and {head.dtype})")
    rows, dim = hidden.shape
    if head.shape[1] != dim:
        _refuse(f"hidden has rows of {dim}, head of {head.shape[1]}")
    target = _vector("target", target, gpu, _INTS, rows)
    h = _Head(hidden.data_ptr(), head.data_ptr(), target.data_ptr(), rows, head.shape[0], dim, hidden.stride(0),
              head.stride(0), _DTYPES[hidden.dtype], _TARGET_BITS[target.dtype], temperature)
    need = _check(lib.dlr_head_logprob_workspace(rows, head.shape[0], dim))
    workspace = torch.empty(need, dtype=torch.uint8, device=hidden.device)
    out, at = _rows(torch.empty((2, rows), dtype=torch.float32, device=hidden.device))
    _check(lib.dlr_head_logprob(gpu, _stream(gpu), C.byref(h), workspace.data_ptr(), need, at, at + 4 * rows))
    return out
