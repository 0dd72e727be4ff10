"""ctypes view of libhccl_amd_model_ops.so (include/hccl_model_ops.h): the operators a training or serving step runs next
to its collectives, over the communicators of this package.

* :func:`token_log_probs` -- log probabilities of given tokens, entropy and top alternatives over a vocabulary that is
  split across the ranks; a collective, every rank receives the results.
* :func:`token_log_probs_grad` -- its gradient with respect to one rank's part of the logits.
* :func:`grad_norm` -- 2-norm over all gradient tensors of all ranks and the factor that clips it; a collective.
* :func:`adamw` -- one AdamW step over many tensors, with states in 32 bits or in FP8 blocks of 256 elements.

Buffers are device pointers (integers, ctypes pointers or anything with ``data_ptr()``), counts are elements, ``stream``
must not be null, and a failing call raises :class:`hccl_amd.HcclError`, as for the collectives; a number that no field of
the C structures holds is refused like any other, and the peers of a collective are released.  Rows of logits and of
their gradient may be any distance apart (``row_stride``); everything else is contiguous.  Drive several ranks from one
thread inside ``with hccl_amd.group():``.  What the arguments mean is written in the header.
"""
import ctypes
import os
import struct

import hccl_amd
from hccl_amd import HcclDataType, HcclError, HcclResult, _as_ptr, _as_stream, check

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libhccl_amd_model_ops.so")
MAX_TOP = 32
STATE_BLOCK = 256

_vp, _u64, _u32, _i32, _f32, _f64 = (ctypes.c_void_p, ctypes.c_uint64, ctypes.c_uint32, ctypes.c_int, ctypes.c_float,
                                     ctypes.c_double)


class TokenLogProbsArgs(ctypes.Structure):
    """HcclAmdTokenLogProbsArgs."""
    _fields_ = [("logits", _vp), ("rowStride", _u64), ("vocabStart", _u64), ("vocabCount", _u64), ("tokenCount", _u64),
                ("tokens", _vp), ("dataType", _i32), ("tokenType", _i32), ("scale", _f32), ("topCount", _u32),
                ("logProbs", _vp), ("logSumExp", _vp), ("entropy", _vp), ("topValues", _vp), ("topIds", _vp),
                ("workspace", _vp), ("workspaceBytes", _u64)]


class TokenLogProbsGradArgs(ctypes.Structure):
    """HcclAmdTokenLogProbsGradArgs."""
    _fields_ = [("logits", _vp), ("rowStride", _u64), ("vocabStart", _u64), ("vocabCount", _u64), ("tokenCount", _u64),
                ("tokens", _vp), ("dataType", _i32), ("tokenType", _i32), ("scale", _f32), ("topCount", _u32),
                ("logSumExp", _vp), ("entropy", _vp), ("gradLogProbs", _vp), ("gradEntropy", _vp), ("topIds", _vp),
                ("gradTopValues", _vp), ("gradLogits", _vp), ("gradRowStride", _u64)]


class NormTensor(ctypes.Structure):
    """HcclAmdNormTensor."""
    _fields_ = [("data", _vp), ("count", _u64), ("dataType", _i32)]


class AdamWTensor(ctypes.Structure):
    """HcclAmdAdamWTensor."""
    _fields_ = [("param", _vp), ("grad", _vp), ("expAvg", _vp), ("expAvgSq", _vp), ("master", _vp), ("expAvgScale", _vp),
                ("expAvgSqScale", _vp), ("count", _u64), ("paramType", _i32), ("gradType", _i32)]


class AdamWConfig(ctypes.Structure):
    """HcclAmdAdamWConfig."""
    _fields_ = [("lr", _f64), ("beta1", _f64), ("beta2", _f64), ("eps", _f64), ("weightDecay", _f64), ("step", _u64),
                ("stepOnDevice", _vp), ("lrOnDevice", _vp), ("clip", _vp), ("stateType", _i32), ("skipNonFinite", _i32)]


def _packer(cls):
    """Packs the fields of the structure `cls`, in order, into the bytes an entry point reads: a fifth of the time the
    ctypes structure itself takes, which counts in calls of a few microseconds."""
    code = {_vp: "Q", _u64: "Q", _u32: "I", _i32: "i", _f32: "f", _f64: "d"}
    packer = struct.Struct("@" + "".join(code[t] for _, t in cls._fields_) + "0Q")
    assert packer.size == ctypes.sizeof(cls)
    return packer.pack


_pack_log_probs = _packer(TokenLogProbsArgs)
_pack_grad = _packer(TokenLogProbsGradArgs)
_pack_config = _packer(AdamWConfig)
_pack_norm = _packer(NormTensor)
_pack_adamw = _packer(AdamWTensor)
_pack_size = struct.Struct("Q").pack
_ANY_STREAM, _ANY_RESULT = ctypes.c_void_p(1), ctypes.c_void_p(4)      # of calls that are refused before they are looked at
_ADAMW_FIELDS = frozenset(("param", "grad", "exp_avg", "exp_avg_sq", "master", "exp_avg_scale", "exp_avg_sq_scale", "count",
                           "param_type", "grad_type"))
_lib = None


def lib():
    """Loads libhccl_amd_model_ops.so; raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    hccl_amd.lib()      # the library it works on
    if not os.path.exists(LIB_PATH):
        raise ImportError("%s is missing: run `make -C hccl_amd/csrc` (or hccl_amd.build()) first" % LIB_PATH)
    _lib = _bind(ctypes.CDLL(LIB_PATH))
    return _lib


def _bind(L):
    """Declares the argument and result types of the library's entry points on the loaded library L."""
    L.HcclAmdTokenLogProbs.argtypes = [_vp, _vp, _vp]
    L.HcclAmdTokenLogProbsWorkspace.argtypes = [_u64, _u64, _u32, ctypes.POINTER(_u64)]
    L.HcclAmdTokenLogProbsGrad.argtypes = [_vp, _vp, _vp]
    L.HcclAmdGradNorm.argtypes = [ctypes.POINTER(NormTensor), _u32, _f32, _f32, _vp, _vp, _u64, _vp, _vp]
    L.HcclAmdGradNormWorkspace.argtypes = [_u64, ctypes.POINTER(_u64)]
    L.HcclAmdAdamW.argtypes = [ctypes.POINTER(AdamWTensor), _u32, _vp, _vp, _vp]
    for name in ("HcclAmdTokenLogProbs", "HcclAmdTokenLogProbsWorkspace", "HcclAmdTokenLogProbsGrad", "HcclAmdGradNorm",
                 "HcclAmdGradNormWorkspace", "HcclAmdAdamW"):
        getattr(L, name).restype = ctypes.c_int
    return L


def _address(buf):
    """_as_ptr as a number; 0 for None."""
    if buf is None:
        return 0
    try:
        return buf.data_ptr()
    except AttributeError:
        return buf if isinstance(buf, int) else _as_ptr(buf).value or 0


def _unfit(where, error, code=0):
    """Raises for a call whose arguments could not be converted: a number that its field does not hold is a parameter error
    like any other bad one, what is no number or buffer at all keeps the error that says so."""
    if isinstance(error, struct.error):
        raise HcclError(code or HcclResult.E_PARA, where) from error
    raise error


def token_log_probs_workspace(token_count, vocab_size, top_count=0):
    """Bytes of workspace a token_log_probs call over `token_count` rows of `vocab_size` entries (all ranks') needs."""
    size = ctypes.c_uint64()
    check(lib().HcclAmdTokenLogProbsWorkspace(token_count, vocab_size, top_count, ctypes.byref(size)),
          "HcclAmdTokenLogProbsWorkspace")
    return size.value


def token_log_probs(hccl_comm, logits, token_count, vocab_start, vocab_count, tokens, log_probs,
                    data_type=HcclDataType.FP32, token_type=HcclDataType.INT64, row_stride=None, scale=1.0, lse=None,
                    entropy=None, top_count=0, top_values=None, top_ids=None, workspace=None, workspace_bytes=0,
                    stream=None):
    """Log probabilities of `tokens` under softmax(scale * logits), whose columns vocab_start .. vocab_start + vocab_count
    this rank holds; every output (log_probs, lse, entropy, top_values, top_ids) may be None."""
    try:
        args = _pack_log_probs(_address(logits), vocab_count if row_stride is None else row_stride, vocab_start, vocab_count,
                               token_count, _address(tokens), data_type, token_type, scale, top_count,
                               _address(log_probs), _address(lse), _address(entropy), _address(top_values),
                               _address(top_ids), _address(workspace), workspace_bytes)
        code = lib().HcclAmdTokenLogProbs(args, hccl_comm, _as_stream(stream))
    except Exception as e:
        # (The library itself raises nothing: it has not been entered.)  The rank takes its place among the
        # collectives all the same, with a call that is refused: its peers return at once.  Without rows no rank takes one.
        rows = 0 if isinstance(token_count, int) and token_count == 0 else 2 ** 64 - 1
        args = _pack_log_probs(0, 0, 0, 0, rows, 0, HcclDataType.FP32, HcclDataType.INT64, 1.0, 0, 0, 0, 0, 0, 0, 0, 0)
        _unfit("HcclAmdTokenLogProbs", e, lib().HcclAmdTokenLogProbs(args, hccl_comm, _ANY_STREAM))
    return check(code, "HcclAmdTokenLogProbs")


def token_log_probs_grad(hccl_comm, logits, token_count, vocab_start, vocab_count, tokens, lse, grad_log_probs, grad_logits,
                         data_type=HcclDataType.FP32, token_type=HcclDataType.INT64, row_stride=None,
                         grad_row_stride=None, scale=1.0, entropy=None, grad_entropy=None, top_count=0, top_ids=None,
                         grad_top_values=None, stream=None):
    """Writes the gradient with respect to this rank's part of the logits to `grad_logits` (which may be the logits
    themselves); local to the rank."""
    try:
        args = _pack_grad(_address(logits), vocab_count if row_stride is None else row_stride, vocab_start, vocab_count,
                          token_count, _address(tokens), data_type, token_type, scale, top_count, _address(lse),
                          _address(entropy), _address(grad_log_probs), _address(grad_entropy), _address(top_ids),
                          _address(grad_top_values), _address(grad_logits),
                          vocab_count if grad_row_stride is None else grad_row_stride)
    except struct.error as e:
        _unfit("HcclAmdTokenLogProbsGrad", e)
    return check(lib().HcclAmdTokenLogProbsGrad(args, hccl_comm, _as_stream(stream)), "HcclAmdTokenLogProbsGrad")


def norm_tensors(tensors):
    """The array grad_norm takes, from (buffer, count, data type) triples; it can be kept while the buffers stay."""
    try:
        items = [_pack_norm(_address(buf), count, data_type) for buf, count, data_type in tensors]
    except struct.error as e:
        _unfit("norm_tensors", e)
    return (NormTensor * len(items)).from_buffer_copy(b"".join(items))


def grad_norm_workspace(tensor_count):
    """Bytes of workspace a grad_norm call over `tensor_count` tensors, all ranks' together, needs."""
    size = ctypes.c_uint64()
    check(lib().HcclAmdGradNormWorkspace(tensor_count, ctypes.byref(size)), "HcclAmdGradNormWorkspace")
    return size.value


def grad_norm(hccl_comm, tensors, max_norm, result, scale=1.0, workspace=None, workspace_bytes=0, stream=None):
    """result[0] = |scale| * 2-norm of all tensors of all ranks, result[1] = scale * the factor that brings it to
    `max_norm` (max_norm <= 0: no clipping).  `tensors`: what norm_tensors returned, or its argument."""
    try:
        if not (isinstance(tensors, ctypes.Array) and tensors._type_ is NormTensor):
            tensors = norm_tensors(tensors)
        _pack_size(workspace_bytes)      # (ctypes would take -1 for a very large workspace)
        code = lib().HcclAmdGradNorm(tensors, len(tensors), max_norm, scale, _as_ptr(result), _as_ptr(workspace),
                                     workspace_bytes, hccl_comm, _as_stream(stream))
    except Exception as e:
        # as in token_log_probs
        _unfit("HcclAmdGradNorm", e, lib().HcclAmdGradNorm(None, 0, float("nan"), 1.0, _ANY_RESULT, None, 0, hccl_comm,
                                                           _ANY_STREAM))
    return check(code, "HcclAmdGradNorm")


def adamw_tensors(tensors):
    """The array adamw takes, from dicts with param, grad, exp_avg, exp_avg_sq, count, param_type, grad_type and, where
    they are wanted, master, exp_avg_scale, exp_avg_sq_scale; it can be kept while the buffers stay."""
    items = []
    for t in tensors:
        if not _ADAMW_FIELDS.issuperset(t):
            raise TypeError("adamw_tensors: unknown fields %s" % sorted(set(t) - _ADAMW_FIELDS))
        try:
            items.append(_pack_adamw(_address(t["param"]), _address(t["grad"]), _address(t["exp_avg"]),
                                     _address(t["exp_avg_sq"]), _address(t.get("master")), _address(t.get("exp_avg_scale")),
                                     _address(t.get("exp_avg_sq_scale")), t["count"], t["param_type"], t["grad_type"]))
        except struct.error as e:
            _unfit("adamw_tensors", e)
    return (AdamWTensor * len(items)).from_buffer_copy(b"".join(items))


def adamw(hccl_comm, tensors, step, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01,
          state_type=HcclDataType.FP32, clip=None, skip_non_finite=False, step_on_device=None, lr_on_device=None,
          stream=None):
    """One AdamW step over all `tensors` (what adamw_tensors returned, or its argument); local to the rank.  `clip` is a
    grad_norm result; `step` counts from 1 (step_on_device: an int64 on the device that is read instead)."""
    if not (isinstance(tensors, ctypes.Array) and tensors._type_ is AdamWTensor):
        tensors = adamw_tensors(tensors)
    try:
        config = _pack_config(lr, beta1, beta2, eps, weight_decay, step, _address(step_on_device), _address(lr_on_device),
                              _address(clip), state_type, 1 if skip_non_finite else 0)
    except struct.error as e:
        _unfit("HcclAmdAdamW", e)
    return check(lib().HcclAmdAdamW(tensors, len(tensors), config, hccl_comm, _as_stream(stream)), "HcclAmdAdamW")
