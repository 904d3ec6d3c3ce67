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
import struct
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


class Heads(C.Structure):
    _fields_ = [("p", vp), ("token", i64), ("head", i64)]


class PackedDims(C.Structure):
    _fields_ = [(n, i32) for n in ("dtype", "nq", "nkv", "head_dim", "n", "Tq", "Tk")] + \
               [("scale", f32), ("q_offsets", vp), ("k_offsets", vp)]


class AdamTensor(C.Structure):
    _fields_ = [(n, vp) for n in ("p", "g", "m", "v", "m_exp", "v_exp", "copy")] + \
               [("n", i64), ("g_dtype", i32), ("copy_dtype", i32)]


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
    # dims and views: addresses of PackedDims and Heads, or their bytes
    "llmt_packed_attention_workspace": (sz, [vp]),
    "llmt_packed_attention": (i32, [vp] * 7 + [sz, vp]),
    "llmt_packed_attention_bwd_workspace": (sz, [vp]),
    "llmt_packed_attention_bwd": (i32, [vp] * 11 + [sz, vp]),
    "llmt_embedding": (i32, [vp, i32, vp, i32, i64, i32, i32, f32, vp, i32, i64, vp]),
    "llmt_embedding_bwd_workspace": (sz, [i32, i32, i32]),
    "llmt_embedding_bwd": (i32, [vp, i32, vp, i32, i64, f32, vp, i32, i64, i32, i32, i32, vp, sz,
                                 vp]),
    "llmt_adamw_update": (i32, [C.POINTER(AdamTensor), i32, i32, C.POINTER(HParams), i32, vp, u64,
                                vp]),
    "llmt_adamw_moments": (i32, [vp, vp, vp, vp, i64, vp, vp, vp]),
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


# ------------------------------------------------------------------ packed sequences

_HEADS = struct.Struct("Pqq")      # a Heads
_PACKED = struct.Struct("7if2P")   # a PackedDims
_HALVES = {}                       # torch.float16 and bfloat16 to the library's codes


def _heads(name, t, shape=None, dtype=None):
    """The bytes of the Heads of a [T, heads, d] tensor (the stride of one token or one head is
    of no account)."""
    at = t.shape
    if shape is not None and (at != shape or t.dtype is not dtype):
        raise LlmtError(f"{name} must be {list(shape)} {dtype} (got {list(at)} {t.dtype})")
    T, heads, d = at
    token, head, one = t.stride()
    if one != 1 and d > 1:
        raise LlmtError(f"{name} must be [T, heads, head_dim] with a last stride of 1")
    if heads < 2:
        head = d
    if T < 2:
        token = (d + 7) // 8 * 8
    return _HEADS.pack(t.data_ptr(), token, head)


def _packed_dims(q, k, v, q_offsets, k_offsets, scale):
    """(the bytes of PackedDims, q's shape and type, k's shape)."""
    import torch
    if not _HALVES:
        _HALVES.update({torch.float16: 1, torch.bfloat16: 2})
    dtype, qs, ks = q.dtype, q.shape, k.shape
    code = _HALVES.get(dtype)
    if code is None or k.dtype is not dtype or v.dtype is not dtype:
        raise LlmtError(f"q, k and v must be float16 or bfloat16 (got {dtype}, {k.dtype}, {v.dtype})")
    if len(qs) != 3 or len(ks) != 3 or v.shape != ks or ks[2] != qs[2]:
        raise LlmtError("q must be [Tq, nq, head_dim], k and v [Tk, nkv, head_dim]")
    _expect("q_offsets", q_offsets, torch.int32, None)
    n = q_offsets.shape[0] - 1
    if n < 1:
        raise LlmtError("offsets must be [n + 1] with n >= 1")
    if k_offsets is None:
        k_offsets = q_offsets
        if ks[0] != qs[0]:
            raise LlmtError(f"without k_offsets q and k are the same tokens (got {qs[0]} and {ks[0]})")
    else:
        _expect("k_offsets", k_offsets, torch.int32, n + 1)
    _sizes("tokens, heads", n + 1, *qs, *ks)
    if scale is None:
        scale = (qs[2] or 1) ** -0.5
    try:
        return _PACKED.pack(code, qs[1], ks[1], qs[2], n, qs[0], ks[0], scale, q_offsets.data_ptr(),
                            k_offsets.data_ptr()), qs, ks, dtype
    except (OverflowError, struct.error):
        raise LlmtError(f"scale must be positive and finite in fp32 (got {scale})") from None


def packed_attention(q, k, v, q_offsets, k_offsets=None, scale=None, out=None, stream=None):
    """Causal attention with grouped heads over packed sequences (llmt_packed_attention): q [Tq,
    nq, d], k and v [Tk, nkv, d] fp16 or bf16, d 64 or 128, views of any strides with d
    contiguous; sequence s has queries q_offsets[s] .. q_offsets[s + 1] - 1 and keys k_offsets[s]
    .. (int32 [n + 1]; None: the queries').  Its last query sees all of its keys.  scale None: 1 /
    sqrt(d).  Returns (o like q, lse fp32 [Tq, nq]); 0 and -inf where a query has no keys."""
    import torch
    with _On("q k v q_offsets k_offsets out", (q, k, v, q_offsets, k_offsets, out), stream) as on:
        dims, qs, ks, dtype = _packed_dims(q, k, v, q_offsets, k_offsets, scale)
        o = q.new_empty(qs) if out is None else out
        lse = q.new_empty(qs[:2], dtype=torch.float32)
        L = lib()
        need = L.llmt_packed_attention_workspace(dims)
        ws = q.new_empty(need, dtype=torch.uint8) if need else None
        check(L.llmt_packed_attention(dims, _heads("q", q), _heads("k", k), _heads("v", v),
                                      _heads("out", o, qs, dtype), lse.data_ptr(), _at(ws), need,
                                      on.raw))
    return o, lse


def packed_attention_bwd(q, k, v, o, lse, dout, q_offsets, k_offsets=None, scale=None, out=None,
                         stream=None):
    """Gradients (dq, dk, dv) of packed_attention in q's type, from its o and lse and dout, the
    gradient of o.  out: the three tensors to write, of any strides (parts of a fused
    projection's gradient)."""
    import torch
    dq = dk = dv = None
    if out is not None:
        if len(out) != 3 or any(t is None for t in out):
            raise LlmtError("out must be the three tensors dq, dk and dv")
        dq, dk, dv = out
    with _On("q k v o lse dout q_offsets k_offsets dq dk dv",
             (q, k, v, o, lse, dout, q_offsets, k_offsets, dq, dk, dv), stream) as on:
        dims, qs, ks, dtype = _packed_dims(q, k, v, q_offsets, k_offsets, scale)
        _expect("lse", lse, torch.float32, qs[0], qs[1])
        if out is None:
            dq, dk, dv = q.new_empty(qs), k.new_empty(ks), v.new_empty(ks)
        L = lib()
        need = L.llmt_packed_attention_bwd_workspace(dims)
        ws = q.new_empty(need, dtype=torch.uint8) if need else None
        check(L.llmt_packed_attention_bwd(
            dims, _heads("q", q), _heads("k", k), _heads("v", v), _heads("o", o, qs, dtype),
            lse.data_ptr(), _heads("dout", dout, qs, dtype), _heads("dq", dq, qs, dtype),
            _heads("dk", dk, ks, dtype), _heads("dv", dv, ks, dtype), _at(ws), need, on.raw))
    return dq, dk, dv


def embedding(tokens, weight, scale=1.0, out_dtype=None, stream=None):
    """scale weight[tokens] (llmt_embedding): tokens int32 of any shape, weight [V, H] fp32, fp16
    or bf16 (rows may be strided); zeros where a token is outside [0, V).  out_dtype None: the
    weight's.  Returns [*tokens.shape, H]."""
    import torch
    with _On("tokens weight", (tokens, weight), stream) as on:
        if tokens.dtype != torch.int32 or not tokens.is_contiguous():
            raise LlmtError("tokens must be contiguous int32")
        wd = _logits_dtype("weight", weight)
        V, H = weight.shape
        T = tokens.numel()
        _sizes("tokens, V, H", T, V, H)
        out = weight.new_empty((*tokens.shape, H), dtype=out_dtype)
        check(lib().llmt_embedding(tokens.data_ptr(), T, weight.data_ptr(), wd, _ld(weight), V, H,
                                   scale, out.data_ptr(), _type_code("out_dtype", out.dtype), H,
                                   on.raw))
    return out


def embedding_bwd(tokens, dout, dweight, scale=1.0, accumulate=False, stream=None):
    """The table's gradient (llmt_embedding_bwd), written into dweight [V, H] fp32, fp16 or bf16
    (rows may be strided) or, with accumulate, added to it; tokens int32 of any shape, dout
    [*tokens.shape, H].  Sums are in the order of the tokens' positions.  Returns dweight."""
    import torch
    with _On("tokens dout dweight", (tokens, dout, dweight), stream) as on:
        if tokens.dtype != torch.int32 or not tokens.is_contiguous():
            raise LlmtError("tokens must be contiguous int32")
        wd = _logits_dtype("dweight", dweight)
        V, H = dweight.shape
        T = tokens.numel()
        if dout.shape != (*tokens.shape, H):
            raise LlmtError(f"dout must be {[*tokens.shape, H]} (got {list(dout.shape)})")
        ldd = H
        if not dout.is_contiguous():
            if dout.dim() != 2 or (H > 1 and dout.stride(1) != 1):
                raise LlmtError("dout must be contiguous, or [T, H] with a column stride of 1")
            ldd = _ld(dout)
        _sizes("tokens, V, H", T, V, H)
        L = lib()
        need = L.llmt_embedding_bwd_workspace(T, V, H)
        ws = dweight.new_empty(need, dtype=torch.uint8) if need else None
        check(L.llmt_embedding_bwd(tokens.data_ptr(), T, dout.data_ptr(),
                                   _type_code("dout", dout.dtype), ldd, scale, dweight.data_ptr(), wd,
                                   _ld(dweight), V, H, int(accumulate), _at(ws), need, on.raw))
    return dweight


def _type_code(name, dtype):
    import torch
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}.get(dtype)
    if code is None:
        raise LlmtError(f"{name} must be float32, float16 or bfloat16 (got {dtype})")
    return code


class AdamState(NamedTuple):
    """Moments of one tensor of n elements: fp32 m and v [n] (m_exp and v_exp None), or 8-bit codes
    uint8 [n] with a byte for each block of 256 elements."""
    m: object
    v: object
    m_exp: object
    v_exp: object


def adamw_state(p, bits=32) -> AdamState:
    """Moments of 0 for a tensor p, of 32 or 8 bits."""
    import torch
    n = p.numel()
    if bits == 32:
        return AdamState(*(torch.zeros(n, dtype=torch.float32, device=p.device) for _ in range(2)),
                         None, None)
    if bits != 8:
        raise LlmtError(f"bits must be 32 or 8 (got {bits})")
    m, v = (torch.zeros(n, dtype=torch.uint8, device=p.device) for _ in range(2))
    return AdamState(m, v, *(torch.zeros(-(-n // 256), dtype=torch.uint8, device=p.device)
                             for _ in range(2)))


class AdamTensors:
    """A list of tensors for adamw_update: parameters fp32, gradients of any type, states (of
    adamw_state, all of one width) and, where given, 16-bit working copies (or None for some);
    contiguous, all on one device.  Keeps their memory: a program makes one list and updates it
    every step.  A tensor that is given other memory later (``p.data = ..``, gradients set to None
    and made anew) needs set_grads or a new list."""

    def __init__(self, params, grads, states, copies=None):
        import torch
        k = len(params)
        copies = [None] * k if copies is None else list(copies)
        if not (len(grads) == len(states) == len(copies) == k):
            raise LlmtError(f"{k} params, {len(grads)} grads, {len(states)} states, {len(copies)} "
                            "copies")
        self.tensors = []          # of every descriptor, in its order
        self.table = (AdamTensor * k)()
        widths = {8 if s[2] is not None else 32 for s in states}
        if len(widths) > 1:
            raise LlmtError("states must be all of 32 or all of 8 bits")
        self.bits = widths.pop() if widths else 32
        self.device = None
        for i, (p, g, s, c) in enumerate(zip(params, grads, states, copies)):
            n = p.numel()
            code = torch.uint8 if self.bits == 8 else torch.float32
            nb = -(-n // 256)
            for name, t, dtype, size in (
                    ("params", p, torch.float32, n), ("grads", g, None, n), ("states' m", s[0], code, n),
                    ("states' v", s[1], code, n), ("states' m_exp", s[2], torch.uint8, nb),
                    ("states' v_exp", s[3], torch.uint8, nb), ("copies", c, None, n)):
                self._check(f"{name}[{i}]", t, dtype, size, self.bits, name)
            if c is not None and c.dtype not in (torch.float16, torch.bfloat16):
                raise LlmtError(f"copies[{i}] must be float16 or bfloat16 (got {c.dtype})")
            self.table[i] = AdamTensor(
                p.data_ptr(), g.data_ptr(), s[0].data_ptr(), s[1].data_ptr(), _at(s[2]), _at(s[3]),
                _at(c), n, _type_code(f"grads[{i}]", g.dtype),
                0 if c is None else _type_code("copies", c.dtype))
            self.tensors.append([None if t is None else t.detach() for t in (p, g, *s, c)])

    def _check(self, name, t, dtype, size, bits, kind):
        import torch
        if t is None:
            if kind == "copies" or (bits == 32 and kind.endswith("exp")):
                return
            raise LlmtError(f"{name} is missing")
        if not isinstance(t, torch.Tensor) or t.get_device() < 0:
            raise LlmtError(f"{name} must be a device tensor")
        if self.device is None:
            self.device = t.get_device()
        if t.get_device() != self.device:
            raise LlmtError(f"{name} is on device {t.get_device()}, other tensors on {self.device}")
        if dtype is not None and t.dtype != dtype:
            raise LlmtError(f"{name} must be {dtype} (got {t.dtype})")
        if t.numel() != size or not t.is_contiguous():
            raise LlmtError(f"{name} must be contiguous with {size} elements (got {t.numel()})")

    def set_grads(self, grads):
        """Other gradients for the same parameters."""
        if len(grads) != len(self.tensors):
            raise LlmtError(f"{len(grads)} grads for {len(self.tensors)} params")
        for i, g in enumerate(grads):
            self._check(f"grads[{i}]", g, None, self.table[i].n, self.bits, "grads")
            _type_code(f"grads[{i}]", g.dtype)
        for i, g in enumerate(grads):
            self.table[i].g = g.data_ptr()
            self.table[i].g_dtype = _type_code("grads", g.dtype)
            self.tensors[i][1] = g.detach()


def adamw_update(tensors: AdamTensors, hp: HParams, step: int, grad_scale=None, seed=0,
                 stream=None):
    """One AdamW step in place over all tensors (llmt_adamw_update).  grad_scale fp32 [1] on the
    device: a factor of the gradients (clipping, a loss scale's inverse).  seed: of the 8-bit
    moments' rounding; the step's number enters its draws too.  A captured call keeps its step and
    its tensors."""
    import torch
    if not tensors.tensors:
        return
    first = tensors.tensors[0][0]
    with _On("params grad_scale", (first, grad_scale), stream) as on:
        _expect("grad_scale", grad_scale, torch.float32, 1)
        if stream is not None:
            on.inputs = [t for row in tensors.tensors for t in row] + [grad_scale]
        check(lib().llmt_adamw_update(tensors.table, len(tensors.tensors), tensors.bits, hp, step,
                                      _at(grad_scale), seed & (2 ** 64 - 1), on.raw))


def adamw_moments(state, stream=None):
    """(m, v) in fp32 of a state of adamw_state: its own tensors at 32 bits, what the codes stand
    for at 8."""
    import torch
    m, v, me, ve = state
    if me is None:
        return m, v
    with _On("m v m_exp v_exp", (m, v, me, ve), stream) as on:
        n = m.numel()
        for name, t, size in (("m", m, n), ("v", v, n), ("m_exp", me, -(-n // 256)),
                              ("v_exp", ve, -(-n // 256))):
            _expect(name, t, torch.uint8, size)
        m32, v32 = (torch.empty(n, dtype=torch.float32, device=m.device) for _ in range(2))
        check(lib().llmt_adamw_moments(m.data_ptr(), v.data_ptr(), me.data_ptr(), ve.data_ptr(), n,
                                       m32.data_ptr(), v32.data_ptr(), on.raw))
    return m32, v32


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
