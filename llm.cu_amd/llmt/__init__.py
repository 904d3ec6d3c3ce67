"""ctypes binding of libllmt.so (include/llmt.h) for tests and the bench.

Tensors are torch tensors used only as device-memory plumbing: every
computation happens in libllmt.so's HIP kernels.  ``lib()`` raises if the
shared library has not been built (``python llm.cu_amd/build.py``); there is
no fallback path.
"""
from __future__ import annotations

import ctypes as C
import os
import re
from pathlib import Path
from typing import NamedTuple

HERE = Path(__file__).resolve().parent
PKG = HERE.parent
ROOT = PKG.parent
# Always the in-tree build: tests and the bench must measure the library
# built from this tree, so an override of the path is refused outright.
if os.environ.get("LLMT_LIB"):
    raise ImportError("LLMT_LIB is set; llmt loads only the in-tree llm.cu_amd/libllmt.so "
                      "(unset LLMT_LIB)")
LIB_PATH = PKG / "libllmt.so"
HEADER = ROOT / "include" / "llmt.h"

vp, i32, f32, sz, u64 = C.c_void_p, C.c_int, C.c_float, C.c_size_t, C.c_uint64
i64 = C.c_longlong
fp = C.POINTER(C.c_float)

LLMT_OK, LLMT_ERR_ARG, LLMT_ERR_HIP, LLMT_ERR_IO, LLMT_ERR_STATE = 0, -1, -2, -3, -4
PROJ = {"wq": 0, "wk": 1, "wv": 2, "wo": 3}
KIND = {"param": 0, "grad": 1, "m": 2, "v": 3}


class LlmtError(RuntimeError):
    pass


class Dims(C.Structure):
    _fields_ = [(n, i32) for n in ("hidden", "n_layers", "n_heads", "n_kv_heads", "head_dim",
                                   "intermediate", "vocab", "rank")] + \
               [(n, f32) for n in ("alpha", "eps", "theta")]


class HParams(C.Structure):
    _fields_ = [(n, f32) for n in ("lr", "beta1", "beta2", "eps", "wd")]


class PrefParams(C.Structure):
    _fields_ = [("kind", i32), ("average", i32)] + \
               [(n, f32) for n in ("beta", "label_smoothing", "margin")]


class PolicyParams(C.Structure):
    _fields_ = [("mean", i32), ("adv_per_sequence", i32)] + \
               [(n, f32) for n in ("clip_low", "clip_high", "kl_coef", "entropy_coef")]


class MuonParams(C.Structure):
    _fields_ = [(n, f32) for n in ("lr", "momentum", "wd", "eps")] + \
               [(n, i32) for n in ("steps", "nesterov", "scale")]


# name -> (restype, argtypes)
_PROTOS = {
    "llmt_last_error": (C.c_char_p, []),
    "llmt_dims_qwen3_1_7b": (None, [C.POINTER(Dims)]),
    "llmt_gemm_f16": (i32, [vp, i32, vp, i32, vp, i32, i32, i32, i32, vp]),
    "llmt_gemm_i8": (i32, [vp, i32, vp, i32, vp, vp, i32, i32, i32, i32, vp]),
    "llmt_quantize_rows_i8": (i32, [vp, i32, i32, vp, vp, vp]),
    "llmt_cross_entropy": (i32, [vp, vp, i32, i32, i32, vp, vp, vp, vp]),
    "llmt_lm_head_ce": (i32, [vp, vp, vp, i32, i32, i32, i32, vp, vp, vp, vp]),
    "llmt_attention_fwd": (i32, [vp, vp, vp, vp, vp, i32, i32, i32, i32, vp]),
    "llmt_attention_bwd": (i32, [vp, vp, vp, vp, vp, vp, vp, vp, vp, i32, i32, i32, i32, vp]),
    "llmt_attention_block_bwd": (i32, [vp, vp, vp, vp, vp, vp, vp, vp, vp, i32, i32, i32, i32,
                                       f32, f32, vp]),
    "llmt_token_logprobs_workspace": (sz, [i32, i32, i32]),
    "llmt_token_logprobs": (i32, [vp, i32, i64, vp, i32, i32, f32, vp, vp, vp, vp, sz, vp]),
    "llmt_token_logprobs_bwd": (i32, [vp, i32, i64, vp, vp, vp, vp, vp, i32, i32, f32, vp, i64,
                                      vp]),
    "llmt_forward_logprobs": (i32, [vp, vp, vp, i32, vp]),
    "llmt_backward_logprobs": (i32, [vp, vp]),
    "llmt_preference_loss": (i32, [vp, vp, vp, vp, i32, i32, C.POINTER(PrefParams), vp, vp, vp,
                                   vp, vp]),
    "llmt_policy_loss_workspace": (sz, [i32, i32]),
    "llmt_policy_loss": (i32, [vp] * 7 + [i32, i32, C.POINTER(PolicyParams)] + [vp] * 5 + [sz, vp]),
    "llmt_orthogonalize_workspace": (sz, [i32, i32, i32]),
    "llmt_orthogonalize": (i32, [vp, i64, i64, vp, i64, i64, i32, i32, i32, i32, f32, vp, sz, vp]),
    "llmt_muon_update_workspace": (sz, [i32, i32, C.POINTER(i32), C.POINTER(i32)]),
    "llmt_muon_update": (i32, [vp, vp, vp, i32, i32, C.POINTER(i32), C.POINTER(i32),
                               C.POINTER(MuonParams), vp, sz, vp]),
    "llmt_muon": (i32, [vp, C.POINTER(MuonParams)]),
    "llmt_ctx_create": (i32, [C.POINTER(Dims), i32, i32, i32, vp, C.POINTER(vp)]),
    "llmt_ctx_destroy": (i32, [vp]),
    "llmt_ctx_device_bytes": (sz, [vp]),
    "llmt_set_layer_f16": (i32, [vp, i32] + [vp] * 11),
    "llmt_set_layer_i8": (i32, [vp, i32, C.POINTER(vp), C.POINTER(vp), vp, vp, vp, vp]),
    "llmt_set_embed_f16": (i32, [vp, vp, vp]),
    "llmt_set_lm_head_f16": (i32, [vp, vp]),
    "llmt_load_weights_dir": (i32, [vp, C.c_char_p]),
    "llmt_lora_numel": (sz, [vp]),
    "llmt_lora_offset": (sz, [vp, i32, i32, i32]),
    "llmt_lora_copy": (i32, [vp, i32, vp, i32]),
    "llmt_lora_save": (i32, [vp, C.c_char_p, i32]),
    "llmt_lora_load": (i32, [vp, C.c_char_p, i32]),
    "llmt_lora_save_state": (i32, [vp, C.c_char_p, i32]),
    "llmt_lora_load_state": (i32, [vp, C.c_char_p, i32]),
    "llmt_lora_init": (i32, [vp, u64, f32, f32]),
    "llmt_step": (i32, [vp, vp, vp, i32, C.POINTER(HParams), i32, fp]),
    "llmt_forward_backward": (i32, [vp, vp, vp, i32, fp]),
    "llmt_set_graph": (i32, [vp, i32]),
    "llmt_logits": (vp, [vp]),
    "llmt_layer_in": (vp, [vp, i32]),
    "llmt_layer_forward": (i32, [vp, i32, vp, vp, i32]),
    "llmt_layer_backward": (i32, [vp, i32, vp, vp, i32]),
    "llmt_adamw": (i32, [vp, C.POINTER(HParams), i32]),
    "llmt_head_ce": (i32, [vp, vp, vp, i32, fp, vp, vp]),
    "llmt_profile_kernels": (i32, [vp, vp, vp, i32, C.POINTER(HParams), i32, i32, i32,
                                   C.POINTER(C.c_int), C.POINTER(C.c_char_p),
                                   C.POINTER(C.c_int), C.POINTER(C.c_int), fp,
                                   C.POINTER(C.c_double), C.POINTER(C.c_double)]),
}

_lib = None


def lib():
    """Load libllmt.so (raises if it is not built)."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise LlmtError(f"{LIB_PATH} is not built; run python llm.cu_amd/build.py")
        L = C.CDLL(str(LIB_PATH))
        for name, (rt, at) in _PROTOS.items():
            fn = getattr(L, name, None)
            if fn is None:
                continue
            fn.restype = rt
            fn.argtypes = at
        _lib = L
    return _lib


def header_functions():
    """Every function name declared in include/llmt.h."""
    txt = HEADER.read_text()
    txt = re.sub(r"/\*.*?\*/", "", txt, flags=re.S)
    names = re.findall(r"^\s*(?:const\s+)?[A-Za-z_][\w\s\*]*?[\s\*](\w+)\s*\(", txt, flags=re.M)
    return sorted(set(n for n in names if n not in ("if", "while", "for", "return", "sizeof")))


def check(rc: int):
    if rc != LLMT_OK:
        raise LlmtError(f"llmt error {rc}: {lib().llmt_last_error().decode()}")


def ptr(t):
    """Device (or host) address of a tensor, or None."""
    return None if t is None else C.c_void_p(t.data_ptr())


def stream_ptr(stream=None):
    import torch
    s = stream if stream is not None else torch.cuda.current_stream()
    return C.c_void_p(s.cuda_stream)


def qwen3_dims() -> Dims:
    d = Dims()
    lib().llmt_dims_qwen3_1_7b(C.byref(d))
    return d


def make_dims(o) -> Dims:
    """Dims from an object with the oracle's Dims attribute names."""
    return Dims(o.hidden, o.n_layers, o.n_heads, o.n_kv_heads, o.head_dim, o.intermediate,
                o.vocab, o.rank, float(o.alpha), float(o.eps), float(o.theta))


# ------------------------------------------------------------------ operators

def gemm_f16(A, B, out=None, stream=None):
    """out[M, N] fp32 = A[M, K] @ B[N, K]^T with fp16 inputs."""
    import torch
    M, K = A.shape
    N = B.shape[0]
    if out is None:
        out = torch.empty(M, N, dtype=torch.float32, device=A.device)
    check(lib().llmt_gemm_f16(ptr(A), A.stride(0), ptr(B), B.stride(0), ptr(out), out.stride(0),
                              M, N, K, stream_ptr(stream)))
    return out


def gemm_i8(A, q, scale16, out=None, stream=None):
    import torch
    M, K = A.shape
    N = q.shape[0]
    if out is None:
        out = torch.empty(M, N, dtype=torch.float32, device=A.device)
    check(lib().llmt_gemm_i8(ptr(A), A.stride(0), ptr(q), q.stride(0), ptr(scale16), ptr(out),
                             out.stride(0), M, N, K, stream_ptr(stream)))
    return out


def quantize_rows_i8(w, stream=None):
    import torch
    rows, cols = w.shape
    q = torch.empty(rows, cols, dtype=torch.int8, device=w.device)
    s = torch.empty(rows, dtype=torch.float32, device=w.device)
    check(lib().llmt_quantize_rows_i8(ptr(w), rows, cols, ptr(q), ptr(s), stream_ptr(stream)))
    return q, s


def cross_entropy(logits, targets, seq_len, want_dlogits=True, stream=None):
    """Returns (loss_mean [1], loss_rows [rows], dlogits or None)."""
    import torch
    rows, V = logits.shape
    dl = torch.empty_like(logits) if want_dlogits else None
    lr = torch.empty(rows, dtype=torch.float32, device=logits.device)
    lm = torch.empty(1, dtype=torch.float32, device=logits.device)
    check(lib().llmt_cross_entropy(ptr(logits), ptr(targets), rows, V, seq_len, ptr(dl), ptr(lr),
                                   ptr(lm), stream_ptr(stream)))
    return lm, lr, dl


# ------------------------------------------------------------------ preferences and rewards

class _On:
    """The device of a call's tensors and its stream, where the outputs and the
    workspace are allocated.  `stream` None is the device's current stream;
    otherwise the inputs are kept from reuse until the stream has passed the
    call.  `raw` is the stream's address."""

    __slots__ = ("inputs", "stream", "ctx", "raw")

    def __init__(self, names, tensors, stream):
        import torch
        index = -1
        for t in tensors:
            if t is not None:
                at = t.get_device() if isinstance(t, torch.Tensor) else -1
                if at != index or at < 0:
                    if index >= 0 or at < 0:
                        name = names.split()[[t is u for u in tensors].index(True)]
                        raise LlmtError(f"{name} must be a device tensor" if at < 0 else
                                        f"{name} is on device {at}, other tensors on {index}")
                    index = at
        self.stream = stream
        if stream is not None:
            if stream.device_index != index:
                raise LlmtError(f"the stream is on {stream.device}, the tensors on device {index}")
            self.inputs = tensors
            self.ctx = torch.cuda.stream(stream)
            self.raw = stream.cuda_stream
        else:
            self.ctx = None if torch._C._cuda_getDevice() == index else torch.cuda.device(index)
            self.raw = torch._C._cuda_getCurrentRawStream(index)

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()
        return self

    def __exit__(self, *exc):
        if self.ctx is not None:
            if self.stream is not None:
                import torch
                if not torch.cuda.is_current_stream_capturing():
                    for t in self.inputs:
                        if t is not None:
                            t.record_stream(self.stream)
            self.ctx.__exit__(*exc)
        return False


def _at(t):
    """The address of a tensor's first element, or None."""
    return None if t is None else t.data_ptr()


def _expect(name, t, dtype, *shape):
    """t, where given, is a contiguous tensor of this type and shape (None: any length)."""
    if t is None or (t.dtype is dtype and t.is_contiguous() and
                     (t.shape == shape or (shape == (None,) and t.dim() == 1))):
        return
    if t.dtype != dtype:
        raise LlmtError(f"{name} must be {dtype} (got {t.dtype})")
    if not t.is_contiguous():
        raise LlmtError(f"{name} must be contiguous")
    raise LlmtError(f"{name} must be {list(shape)} (got {list(t.shape)})")


def _logits_dtype(name, t):
    """The library's code for the type of a [rows, V] tensor with unit column stride."""
    import torch
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}.get(t.dtype)
    if code is None:
        raise LlmtError(f"{name} must be float32, float16 or bfloat16 (got {t.dtype})")
    if t.dim() != 2 or t.shape[1] < 1 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise LlmtError(f"{name} must be [rows, V] with V >= 1 and a column stride of 1")
    return code


def _inverse(temperature):
    if not temperature > 0:
        raise LlmtError(f"temperature must be positive (got {temperature})")
    return 1.0 / temperature


def _ld(t):
    """Elements from row to row (a single row's stride is of no account)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _sizes(names, *sizes):
    """Sizes that the library takes as int (ctypes would pass on their lower 32 bits)."""
    if max(sizes) >= 1 << 31:
        raise LlmtError(f"{names}: {sizes}, each at most 2^31 - 1")


def _byte_mask(mask, T):
    import torch
    if mask is not None:
        _expect("mask", mask, torch.uint8 if mask.dtype is torch.uint8 else torch.bool, T)


def token_logprobs(logits, targets, temperature=1.0, want_entropy=False, stream=None):
    """Log-probabilities of targets int32 [rows] under softmax(logits /
    temperature), logits [rows, V] fp32, fp16 or bf16 (rows may be strided):
    (logp [rows], stats [rows, 2] for token_logprobs_bwd, entropy [rows] or
    None), fp32.  Rows whose target is outside [0, V) are skipped (zeros)."""
    import torch
    with _On("logits targets", (logits, targets), stream) as on:
        dt = _logits_dtype("logits", logits)
        rows, V = logits.shape
        _sizes("rows, V", rows, V)
        _expect("targets", targets, torch.int32, rows)
        logp = logits.new_empty(rows, dtype=torch.float32)
        stats = logits.new_empty((rows, 2), dtype=torch.float32)
        ent = torch.empty_like(logp) if want_entropy else None
        L = lib()
        need = L.llmt_token_logprobs_workspace(rows, V, dt)
        ws = logits.new_empty(need, dtype=torch.uint8) if need else None
        check(L.llmt_token_logprobs(logits.data_ptr(), dt, _ld(logits), targets.data_ptr(), rows, V,
                                    _inverse(temperature), logp.data_ptr(), stats.data_ptr(), _at(ent),
                                    _at(ws), need, on.raw))
    return logp, stats, ent


def token_logprobs_bwd(logits, targets, stats, dlogp, entropy=None, dentropy=None,
                       temperature=1.0, out=None, stream=None):
    """The gradient of the logits from those of token_logprobs' logp and,
    where given, its entropy; in the logits' type.  out may be the logits
    themselves (they are overwritten)."""
    import torch
    with _On("logits targets stats dlogp entropy dentropy out",
             (logits, targets, stats, dlogp, entropy, dentropy, out), stream) as on:
        dt = _logits_dtype("logits", logits)
        rows, V = logits.shape
        _sizes("rows, V", rows, V)
        _expect("targets", targets, torch.int32, rows)
        _expect("stats", stats, torch.float32, rows, 2)
        _expect("dlogp", dlogp, torch.float32, rows)
        _expect("entropy", entropy, torch.float32, rows)
        _expect("dentropy", dentropy, torch.float32, rows)
        if out is None:
            out = logits.new_empty((rows, V))
        elif out.shape != logits.shape or _logits_dtype("out", out) != dt:
            raise LlmtError("out must have the logits' shape and type")
        check(lib().llmt_token_logprobs_bwd(logits.data_ptr(), dt, _ld(logits), targets.data_ptr(),
                                            stats.data_ptr(), _at(entropy), dlogp.data_ptr(),
                                            _at(dentropy), rows, V, _inverse(temperature),
                                            out.data_ptr(), _ld(out), on.raw))
    return out


PREF_LOSSES = {"sigmoid": 0, "hinge": 1, "square": 2}
MEANS = {"token": 0, "sequence": 1}


def preference_loss(logp, ref_logp, offsets, loss="sigmoid", beta=0.1, label_smoothing=0.0,
                    margin=0.0, average=False, mask=None, want_grad=True, stream=None):
    """Preference loss of n pairs of sequences (llmt_preference_loss): pair i
    prefers sequence 2 i to 2 i + 1, sequence s being tokens offsets[s] ..
    offsets[s + 1] - 1 of logp and ref_logp (may be None), fp32 [T]; offsets
    int32 [2 n + 1]; mask bool [T] keeps tokens.  loss "square" is (z - 1/2)^2 of
    the beta-scaled z: beta^2 times the identity-preference loss, and so is its
    gradient.  Returns (mean loss [1], losses [n], rewards [2 n], dlogp [T] or
    None)."""
    import torch
    kind = PREF_LOSSES.get(loss)
    if kind is None:
        raise LlmtError(f"loss must be one of {sorted(PREF_LOSSES)} (got {loss!r})")
    with _On("logp ref_logp offsets mask", (logp, ref_logp, offsets, mask), stream) as on:
        _expect("logp", logp, torch.float32, None)
        T = logp.shape[0]
        _expect("ref_logp", ref_logp, torch.float32, T)
        _expect("offsets", offsets, torch.int32, None)
        _byte_mask(mask, T)
        n = offsets.shape[0] // 2
        if n < 1 or offsets.shape[0] != 2 * n + 1:
            raise LlmtError(f"offsets must be [2 n + 1] with n >= 1 (got {list(offsets.shape)})")
        _sizes("T, offsets", T, 2 * n + 1)
        mean, losses, rewards = logp.new_empty(3 * n + 1).split_with_sizes((1, n, 2 * n))
        dlogp = torch.empty_like(logp) if want_grad else None
        p = PrefParams(kind, average, beta, label_smoothing, margin)
        check(lib().llmt_preference_loss(logp.data_ptr(), _at(ref_logp), _at(mask),
                                         offsets.data_ptr(), T, n, p, mean.data_ptr(),
                                         losses.data_ptr(), rewards.data_ptr(), _at(dlogp), on.raw))
    return mean, losses, rewards, dlogp


class PolicyLoss(NamedTuple):
    """loss [1], stats [3] (policy term, KL, share of clipped tokens), and the
    gradients of loss by logp and by entropy [T] (None where not wanted)."""
    loss: object
    stats: object
    dlogp: object
    dentropy: object


def policy_loss(logp, old_logp, advantages, offsets, ref_logp=None, entropy=None, mask=None,
                clip_low=0.2, clip_high=0.2, kl_coef=0.0, entropy_coef=0.0, mean="token",
                per_sequence=False, want_grad=True, stream=None):
    """Clipped policy loss with a KL term (llmt_policy_loss) over n sequences,
    sequence s being tokens offsets[s] .. offsets[s + 1] - 1 of the fp32 [T]
    arrays; advantages [T], or [n] with per_sequence.  old_logp None: ratio 1;
    ref_logp None: no KL term.  Returns a PolicyLoss."""
    import torch
    kind = MEANS.get(mean)
    if kind is None:
        raise LlmtError(f"mean must be one of {sorted(MEANS)} (got {mean!r})")
    with _On("logp old_logp advantages offsets ref_logp entropy mask",
             (logp, old_logp, advantages, offsets, ref_logp, entropy, mask), stream) as on:
        _expect("logp", logp, torch.float32, None)
        T = logp.shape[0]
        _expect("old_logp", old_logp, torch.float32, T)
        _expect("ref_logp", ref_logp, torch.float32, T)
        _expect("entropy", entropy, torch.float32, T)
        _expect("offsets", offsets, torch.int32, None)
        _byte_mask(mask, T)
        n = offsets.shape[0] - 1
        if n < 1:
            raise LlmtError("offsets must be [n + 1] with n >= 1")
        _sizes("T, offsets", T, n + 1)
        _expect("advantages", advantages, torch.float32, n if per_sequence else T)
        L = lib()
        need = L.llmt_policy_loss_workspace(T, n)
        ws = logp.new_empty(need, dtype=torch.uint8) if need else None
        loss, stats = logp.new_empty(1), logp.new_empty(3)
        dlogp = torch.empty_like(logp) if want_grad else None
        dent = torch.empty_like(logp) if want_grad and entropy is not None else None
        p = PolicyParams(kind, per_sequence, clip_low, clip_high, kl_coef, entropy_coef)
        check(L.llmt_policy_loss(logp.data_ptr(), _at(old_logp), _at(ref_logp),
                                 advantages.data_ptr(), _at(entropy), _at(mask), offsets.data_ptr(),
                                 T, n, p, loss.data_ptr(), stats.data_ptr(), _at(dlogp), _at(dent),
                                 _at(ws), need, on.raw))
    return PolicyLoss(loss, stats, dlogp, dent)


# ------------------------------------------------------------------ orthogonalised updates

def orthogonalize(x, steps=5, eps=1e-7, out=None, stream=None):
    """Newton-Schulz orthogonalisation (llmt_orthogonalize) of a matrix [rows,
    cols] or a stack [count, rows, cols], fp32, the short side at most 64; rows
    may be strided.  out may be x itself."""
    import torch
    with _On("x out", (x, out), stream) as on:
        if x.dtype != torch.float32 or x.dim() not in (2, 3) or 0 in x.shape[-2:]:
            raise LlmtError("x must be float32 [rows, cols] or [count, rows, cols]")
        rows, cols = x.shape[-2:]
        count = x.shape[0] if x.dim() == 3 else 1
        _sizes("count, rows, cols", count, rows, cols)
        if out is None:
            out = x.new_empty(x.shape)
        elif out.shape != x.shape or out.dtype != torch.float32:
            raise LlmtError("out must have x's shape and type")

        def strides(name, t):  # of one row or one matrix the stride is of no account
            if cols > 1 and t.stride(-1) != 1:
                raise LlmtError(f"{name} must have a column stride of 1")
            ld = t.stride(-2) if rows > 1 else cols
            return (t.stride(0) if count > 1 else rows * ld), ld

        (sx, ldx), (so, ldo) = strides("x", x), strides("out", out)
        L = lib()
        need = L.llmt_orthogonalize_workspace(count, rows, cols)
        ws = x.new_empty(need, dtype=torch.uint8) if need else None
        check(L.llmt_orthogonalize(x.data_ptr(), sx, ldx, out.data_ptr(), so, ldo, count, rows,
                                   cols, steps, eps, _at(ws), need, on.raw))
    return out


MUON_SCALES = {"rms": 0, "shape": 1}


def muon_hparams(lr=2e-3, momentum=0.95, wd=0.01, eps=1e-7, steps=5, nesterov=True,
                 scale="rms") -> MuonParams:
    """Muon's hyper-parameters (llmt_muon_update)."""
    if scale not in MUON_SCALES:
        raise LlmtError(f"scale must be one of {sorted(MUON_SCALES)} (got {scale!r})")
    return MuonParams(lr, momentum, wd, eps, steps, int(nesterov), MUON_SCALES[scale])


def muon_update(p, g, m, shapes, hp: MuonParams, stream=None):
    """One Muon step in place on flat fp32 arenas p and m from the gradients g:
    layers of the matrices `shapes` [(rows, cols), ..] one behind another."""
    import torch
    with _On("p g m", (p, g, m), stream) as on:
        _expect("p", p, torch.float32, None)
        n = p.shape[0]
        _expect("g", g, torch.float32, n)
        _expect("m", m, torch.float32, n)
        per = sum(r * c for r, c in shapes)
        if per < 1 or n < 1 or n % per:
            raise LlmtError(f"the arena's {n} elements are not whole layers of {per}")
        k = len(shapes)
        rows, cols = zip(*shapes)
        _sizes("layers, rows, cols", n // per, *rows, *cols)
        rows, cols = (i32 * k)(*rows), (i32 * k)(*cols)
        L = lib()
        need = L.llmt_muon_update_workspace(n // per, k, rows, cols)
        ws = p.new_empty(need, dtype=torch.uint8) if need else None
        check(L.llmt_muon_update(p.data_ptr(), g.data_ptr(), m.data_ptr(), n // per, k, rows, cols,
                                 hp, _at(ws), need, on.raw))


# ------------------------------------------------------------------ training context

PROFILE_CATEGORIES = ("gemm_fwd", "gemm_bwd", "gemm_lm_head", "attention", "row_epilogues",
                      "cross_entropy", "lora_grad", "adamw")


def hparams(lr=3e-4, beta1=0.9, beta2=0.999, eps=1e-8, wd=0.01) -> HParams:
    """AdamW hyper-parameters; defaults are src/train.cu:174-182."""
    return HParams(lr, beta1, beta2, eps, wd)


class Context:
    """One llmt_ctx: frozen weights, adapters, stashes and workspaces of the
    LoRA training step for up to ``max_batch`` sequences of ``seq_len``.

    The library works on ``stream`` (None: one of the context's own, ordered
    with the legacy default stream).  Calls that take or give tensors first
    wait for torch's current stream where it is neither of these, and all end
    with a host synchronisation: tensors are used as they are at the call,
    whatever stream is current."""

    def __init__(self, dims: Dims, max_batch: int, seq_len: int, int8: bool = False, stream=None):
        import torch
        self.h = None
        self.dims = dims
        self.max_batch = max_batch
        self.seq_len = seq_len
        self.logp_rows = 0  # of the last forward_logprobs
        h = vp()
        sp = None if stream is None else C.c_void_p(stream.cuda_stream)
        check(lib().llmt_ctx_create(C.byref(dims), max_batch, seq_len, 1 if int8 else 0, sp,
                                    C.byref(h)))
        self.h = h
        # the stream that needs no wait (0: the legacy default stream)
        self._stream = 0 if stream is None else stream.cuda_stream
        self._device = torch.cuda.current_device() if stream is None else stream.device_index

    def _follow(self):
        """Puts the context's stream behind torch's current one."""
        import torch
        if torch.cuda.is_initialized():
            at = torch.cuda.current_stream(self._device)
            if at.cuda_stream != self._stream:
                at.synchronize()

    def close(self):
        if self.h:
            lib().llmt_ctx_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def device_bytes(self) -> int:
        return lib().llmt_ctx_device_bytes(self.h)

    # -- weights
    def set_layer_f16(self, layer, wq, wk, wv, wo, w_gate, w_up, w_down, attn_norm, ffn_norm,
                      q_norm, k_norm):
        self._follow()
        check(lib().llmt_set_layer_f16(self.h, layer, *(ptr(t) for t in (
            wq, wk, wv, wo, w_gate, w_up, w_down, attn_norm, ffn_norm, q_norm, k_norm))))

    def set_layer_i8(self, layer, qs, scales16, attn_norm, ffn_norm, q_norm, k_norm):
        self._follow()
        qa = (vp * 7)(*(t.data_ptr() for t in qs))
        sa = (vp * 7)(*(t.data_ptr() for t in scales16))
        check(lib().llmt_set_layer_i8(self.h, layer, qa, sa, ptr(attn_norm), ptr(ffn_norm),
                                      ptr(q_norm), ptr(k_norm)))

    def set_embed_f16(self, embed, final_norm):
        self._follow()
        check(lib().llmt_set_embed_f16(self.h, ptr(embed), ptr(final_norm)))

    def set_lm_head_f16(self, lm_head):
        """An untied lm_head [V, H] fp16 (llmt_set_lm_head_f16)."""
        self._follow()
        check(lib().llmt_set_lm_head_f16(self.h, ptr(lm_head)))

    def load_weights_dir(self, path):
        check(lib().llmt_load_weights_dir(self.h, str(path).encode()))

    # -- adapters
    @property
    def lora_numel(self) -> int:
        return lib().llmt_lora_numel(self.h)

    def lora_offset(self, layer, proj, is_b) -> int:
        return lib().llmt_lora_offset(self.h, layer, PROJ[proj] if isinstance(proj, str) else proj,
                                      int(is_b))

    def lora_set(self, kind: str, flat):
        """Copy a flat fp32 tensor (device or host) into an arena."""
        flat = flat.contiguous()
        assert flat.numel() == self.lora_numel and flat.dtype.is_floating_point
        self._follow()
        check(lib().llmt_lora_copy(self.h, KIND[kind], ptr(flat), 1))

    def lora_get(self, kind: str, device="cuda"):
        import torch
        out = torch.empty(self.lora_numel, dtype=torch.float32, device=device)
        self._follow()
        check(lib().llmt_lora_copy(self.h, KIND[kind], ptr(out), 0))
        return out

    def lora_init(self, seed: int, a_std: float, b_std: float):
        check(lib().llmt_lora_init(self.h, seed, a_std, b_std))

    def lora_save(self, path, step: int):
        check(lib().llmt_lora_save(self.h, str(path).encode(), step))

    def lora_load(self, path, step: int):
        check(lib().llmt_lora_load(self.h, str(path).encode(), step))

    def lora_save_state(self, path, step: int):
        """AdamW moments, or Muon's momentum, to <path>/lora_step{step}_adamw.bin
        (for resuming with the same optimiser)."""
        check(lib().llmt_lora_save_state(self.h, str(path).encode(), step))

    def lora_load_state(self, path, step: int):
        check(lib().llmt_lora_load_state(self.h, str(path).encode(), step))

    # -- the step
    def _check_tokens(self, tokens, targets):
        """tokens/targets must be int32 device tensors [B, seq_len] with
        1 <= B <= max_batch, contiguous (the library copies B * seq_len ids
        from each pointer; the step graph repeats that copy on every replay)."""
        import torch
        for name, t in (("tokens", tokens), ("targets", targets)):
            if not isinstance(t, torch.Tensor):
                raise LlmtError(f"{name} must be a torch tensor")
            if t.dtype != torch.int32:
                raise LlmtError(f"{name} must be int32 (got {t.dtype})")
            if not t.is_cuda:
                raise LlmtError(f"{name} must be a device tensor")
            if not t.is_contiguous():
                raise LlmtError(f"{name} must be contiguous")
            if t.dim() != 2 or t.shape[1] != self.seq_len or not 1 <= t.shape[0] <= self.max_batch:
                raise LlmtError(f"{name} must be [B, {self.seq_len}] with 1 <= B <= "
                                f"{self.max_batch} (got {tuple(t.shape)})")
        if tokens.shape != targets.shape:
            raise LlmtError(f"tokens {tuple(tokens.shape)} and targets {tuple(targets.shape)} differ")
        return tokens.shape[0]

    def set_graph(self, enable: bool):
        check(lib().llmt_set_graph(self.h, int(enable)))

    def step(self, tokens, targets, hp: HParams, step: int) -> float:
        B = self._check_tokens(tokens, targets)
        self._follow()
        loss = C.c_float()
        check(lib().llmt_step(self.h, ptr(tokens), ptr(targets), B, C.byref(hp), step,
                              C.byref(loss)))
        return loss.value

    def forward_backward(self, tokens, targets) -> float:
        B = self._check_tokens(tokens, targets)
        self._follow()
        loss = C.c_float()
        check(lib().llmt_forward_backward(self.h, ptr(tokens), ptr(targets), B, C.byref(loss)))
        return loss.value

    def layer_in(self, layer, rows):
        """A copy of the fp32 residual stream [rows, H] at the input of
        `layer` from the last forward (llmt_layer_in)."""
        import torch
        addr = lib().llmt_layer_in(self.h, layer)
        if not addr:
            raise LlmtError(f"llmt_layer_in: no layer {layer}")
        H = self.dims.hidden

        class _View:
            __cuda_array_interface__ = {"shape": (rows, H), "typestr": "<f4",
                                        "data": (addr, False), "version": 3, "strides": None}
        return torch.as_tensor(_View(), device="cuda").clone()

    def logits(self, rows):
        """A copy of the first `rows` rows of the fp32 logits of the last
        forward (llmt_logits)."""
        import torch
        addr = lib().llmt_logits(self.h)
        V = self.dims.vocab

        class _View:
            __cuda_array_interface__ = {"shape": (rows, V), "typestr": "<f4",
                                        "data": (addr, False), "version": 3, "strides": None}
        return torch.as_tensor(_View(), device="cuda").clone()

    def _on_device(self, name, t):
        if t.get_device() != self._device:
            raise LlmtError(f"{name} is on device {t.get_device()}, the context on {self._device}")

    def forward_logprobs(self, tokens, targets):
        """The forward's log-probability of every target, fp32 [B * seq_len]
        (0 where the target is outside [0, V)); backward_logprobs then takes
        the gradient of any function of them (llmt_forward_logprobs)."""
        import torch
        B = self._check_tokens(tokens, targets)
        self._on_device("tokens", tokens)
        self._on_device("targets", targets)
        logp = torch.empty(B * self.seq_len, dtype=torch.float32, device=tokens.device)
        self._follow()
        check(lib().llmt_forward_logprobs(self.h, ptr(tokens), ptr(targets), B, ptr(logp)))
        self.logp_rows = B * self.seq_len
        return logp

    def backward_logprobs(self, dlogp):
        """Adapter gradients into the GRAD arena from the gradient of the last
        forward_logprobs' result (llmt_backward_logprobs)."""
        import torch
        if not (isinstance(dlogp, torch.Tensor) and dlogp.is_cuda):
            raise LlmtError("dlogp must be a device tensor")
        self._on_device("dlogp", dlogp)
        _expect("dlogp", dlogp, torch.float32, self.logp_rows)
        self._follow()
        check(lib().llmt_backward_logprobs(self.h, ptr(dlogp)))

    def muon(self, hp: MuonParams):
        """One Muon step over the adapters from the GRAD arena (llmt_muon)."""
        check(lib().llmt_muon(self.h, C.byref(hp)))

    def head_ce(self, hidden16, targets, want_dlogits=False):
        """C1 on the context's tied embedding: (loss, dlogits or None, dhidden)."""
        import torch
        T = hidden16.shape[0]
        loss = C.c_float()
        dl = torch.empty(T, self.dims.vocab, dtype=torch.float32, device=hidden16.device) \
            if want_dlogits else None
        dh = torch.empty(T, self.dims.hidden, dtype=torch.float32, device=hidden16.device)
        self._follow()
        check(lib().llmt_head_ce(self.h, ptr(hidden16), ptr(targets), T // self.seq_len,
                                 C.byref(loss), ptr(dl), ptr(dh)))
        return loss.value, dl, dh

    def layer_forward(self, layer, x, batch):
        import torch
        y = torch.empty_like(x)
        self._follow()
        check(lib().llmt_layer_forward(self.h, layer, ptr(x), ptr(y), batch))
        return y

    def layer_backward(self, layer, dy, batch):
        import torch
        dx = torch.empty_like(dy)
        self._follow()
        check(lib().llmt_layer_backward(self.h, layer, ptr(dy), ptr(dx), batch))
        return dx

    def profile_kernels(self, tokens, targets, hp: HParams, step: int, reps: int = 5):
        """Per kernel kind of one step (llmt_profile_kernels): a list of dicts
        with name, category, launches (per step), us (average launch
        duration), flops and bytes (per launch; GEMMs only).  The adapters
        advance by one AdamW step."""
        mx = 256
        ns = C.c_int()
        names = (C.c_char_p * mx)()
        cats, nl = (C.c_int * mx)(), (C.c_int * mx)()
        us = (C.c_float * mx)()
        fl, by = (C.c_double * mx)(), (C.c_double * mx)()
        self._follow()
        check(lib().llmt_profile_kernels(self.h, ptr(tokens), ptr(targets),
                                         self._check_tokens(tokens, targets), C.byref(hp), step,
                                         reps, mx, C.byref(ns), names, cats, nl, us, fl, by))
        return [dict(name=names[k].decode(), category=PROFILE_CATEGORIES[cats[k]],
                     launches=nl[k], us=us[k], flops=fl[k], bytes=by[k])
                for k in range(ns.value)]


def flatten_adapters(adapters, attr=("A", "B")):
    """Adapters as list-of-dicts (layer -> proj -> object with A, B) -> one
    flat fp32 tensor in the arena order: layer by layer, q, k, v, o, A then B."""
    import torch
    parts = []
    for d in adapters:
        for p in ("wq", "wk", "wv", "wo"):
            for a in attr:
                parts.append(getattr(d[p], a).reshape(-1).float())
    return torch.cat(parts)


def unflatten_adapters(flat, dims):
    """Inverse of flatten_adapters: list of {proj: (A, B)} tensors (views)."""
    r = dims.rank
    q, kv, hd = dims.n_heads * dims.head_dim, dims.n_kv_heads * dims.head_dim, dims.hidden
    shapes = {"wq": (q, hd), "wk": (kv, hd), "wv": (kv, hd), "wo": (hd, q)}
    out, off = [], 0
    for _ in range(dims.n_layers):
        d = {}
        for p in ("wq", "wk", "wv", "wo"):
            d_out, d_in = shapes[p]
            A = flat[off:off + r * d_in].view(r, d_in)
            off += r * d_in
            B = flat[off:off + d_out * r].view(d_out, r)
            off += d_out * r
            d[p] = (A, B)
        out.append(d)
    assert off == flat.numel()
    return out


def lm_head_ce(hidden16, W16, targets, seq_len, want_dlogits=True, stream=None):
    """Standalone C1: (loss_mean [1], dlogits or None, dhidden [T, H])."""
    import torch
    T, H = hidden16.shape
    V = W16.shape[0]
    lm = torch.empty(1, dtype=torch.float32, device=hidden16.device)
    dl = torch.empty(T, V, dtype=torch.float32, device=hidden16.device) if want_dlogits else None
    dh = torch.empty(T, H, dtype=torch.float32, device=hidden16.device)
    check(lib().llmt_lm_head_ce(ptr(hidden16), ptr(W16), ptr(targets), T, seq_len, H, V, ptr(lm),
                                ptr(dl), ptr(dh), stream_ptr(stream)))
    return lm, dl, dh


def attention_fwd(q, k, v, stream=None):
    """q [B,S,nq,128], k/v [B,S,nkv,128] fp16 -> (o fp16 like q, lse fp32 [B,nq,S])."""
    import torch
    B, S, nq, _ = q.shape
    nkv = k.shape[2]
    o = torch.empty_like(q)
    lse = torch.empty(B, nq, S, dtype=torch.float32, device=q.device)
    check(lib().llmt_attention_fwd(ptr(q), ptr(k), ptr(v), ptr(o), ptr(lse), B, S, nq, nkv,
                                   stream_ptr(stream)))
    return o, lse


def attention_bwd(q, k, v, o, lse, dout32, stream=None):
    """Gradients (fp32) w.r.t. q, k, v of the causal GQA attention."""
    import torch
    B, S, nq, _ = q.shape
    nkv = k.shape[2]
    dq = torch.empty(q.shape, dtype=torch.float32, device=q.device)
    dk = torch.empty(k.shape, dtype=torch.float32, device=q.device)
    dv = torch.empty(v.shape, dtype=torch.float32, device=q.device)
    check(lib().llmt_attention_bwd(ptr(q), ptr(k), ptr(v), ptr(o), ptr(lse), ptr(dout32), ptr(dq),
                                   ptr(dk), ptr(dv), B, S, nq, nkv, stream_ptr(stream)))
    return dq, dk, dv


def attention_block_bwd(q_raw, k_raw, v, q_norm, k_norm, dout16, theta=1e6, eps=1e-6, stream=None):
    """Config C3: QK-norm + RoPE + flash attention forward and backward."""
    import torch
    B, S, nq, _ = q_raw.shape
    nkv = k_raw.shape[2]
    dq = torch.empty(q_raw.shape, dtype=torch.float32, device=q_raw.device)
    dk = torch.empty(k_raw.shape, dtype=torch.float32, device=q_raw.device)
    dv = torch.empty(v.shape, dtype=torch.float32, device=q_raw.device)
    check(lib().llmt_attention_block_bwd(ptr(q_raw), ptr(k_raw), ptr(v), ptr(q_norm), ptr(k_norm),
                                         ptr(dout16), ptr(dq), ptr(dk), ptr(dv), B, S, nq, nkv,
                                         theta, eps, stream_ptr(stream)))
    return dq, dk, dv
