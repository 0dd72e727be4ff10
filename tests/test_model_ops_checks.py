"""CPU tier: the argument checks of the model operators (include/hccl_model_ops.h).  Every call here is refused, or has
nothing to do, before any GPU work; a refused collective keeps its place in the sequence."""
import ctypes
import math
import os
import re
import subprocess
import threading

import pytest

import hccl_amd
from hccl_amd import HcclDataType as DT
from hccl_amd import HcclError, model_ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STREAM = 0x1000        # never dereferenced
A = 0x10000            # a device address that is never touched
OK, PARA, PTR, MEMORY, NOT_SUPPORT, UNAVAIL = 0, 1, 2, 3, 5, 7


@pytest.fixture(scope="module")
def one():
    comms = hccl_amd.comm_init_all(1)
    yield comms[0]
    hccl_amd.comm_destroy(comms[0])


def code(fn, *a, **k):
    try:
        return fn(*a, **k)
    except HcclError as e:
        return e.code


def log_probs(comm, logits=A, token_count=3, vocab_start=0, vocab_count=8, tokens=A, log_probs=A, **k):
    k.setdefault("stream", STREAM)
    return code(model_ops.token_log_probs, comm, logits, token_count, vocab_start, vocab_count, tokens, log_probs, **k)


def grad(comm, logits=A, token_count=3, vocab_start=0, vocab_count=8, tokens=A, lse=A, grad_log_probs=A,
         grad_logits=0x90000, **k):
    k.setdefault("stream", STREAM)
    return code(model_ops.token_log_probs_grad, comm, logits, token_count, vocab_start, vocab_count, tokens, lse,
                grad_log_probs, grad_logits, **k)


def norm(comm, tensors=((A, 4, DT.FP32),), max_norm=1.0, result=A, **k):
    k.setdefault("stream", STREAM)
    return code(model_ops.grad_norm, comm, list(tensors), max_norm, result, **k)


def adamw(comm, change=None, **k):
    t = dict(param=A, grad=A, exp_avg=A, exp_avg_sq=A, count=4, param_type=DT.FP32, grad_type=DT.FP32)
    t.update(change or {})
    k = dict(dict(step=1, lr=1e-3, stream=STREAM), **k)
    return code(model_ops.adamw, comm, [t], **k)


def test_structures_have_the_header_s_layout(tmp_path):
    """Sizes and offsets as the C compiler sees them."""
    structs = {"HcclAmdTokenLogProbsArgs": model_ops.TokenLogProbsArgs,
               "HcclAmdTokenLogProbsGradArgs": model_ops.TokenLogProbsGradArgs, "HcclAmdNormTensor": model_ops.NormTensor,
               "HcclAmdAdamWTensor": model_ops.AdamWTensor, "HcclAmdAdamWConfig": model_ops.AdamWConfig}
    lines = []
    for c, py in structs.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (c, c))
        lines += ['printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (c, f[0], c, f[0]) for f in py._fields_]
    src = tmp_path / "layout.c"
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"hccl_model_ops.h\"\nint main(void) {\n%s\nreturn 0; }\n"
                   % "\n".join(lines))
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Werror", "-I" + os.path.join(ROOT, "include"), str(src), "-o",
                           str(tmp_path / "layout")])
    told = dict(line.split() for line in subprocess.check_output([str(tmp_path / "layout")], text=True).splitlines())
    for c, py in structs.items():
        assert int(told[c]) == ctypes.sizeof(py), c
        for f in py._fields_:
            assert int(told["%s.%s" % (c, f[0])]) == getattr(py, f[0]).offset, (c, f[0])
    header = open(os.path.join(ROOT, "include", "hccl_model_ops.h")).read()
    assert int(re.search(r"HCCL_AMD_MAX_TOP (\d+)", header).group(1)) == model_ops.MAX_TOP
    assert int(re.search(r"HCCL_AMD_STATE_BLOCK (\d+)", header).group(1)) == model_ops.STATE_BLOCK


def test_handles_and_streams(one):
    for call in (log_probs, grad, norm, adamw):
        assert call(one, stream=None) == PTR, call
        assert call(None) == PTR, call
        assert call(ctypes.c_void_p(0x1234560)) == PARA, call      # never issued


def test_nothing_to_do(one):
    assert log_probs(one, token_count=0, logits=None, tokens=None) == OK
    assert grad(one, token_count=0, logits=None) == OK
    assert grad(one, vocab_count=0, logits=None) == OK
    assert code(model_ops.adamw, one, [], step=1, lr=1e-3, stream=STREAM) == OK
    assert adamw(one, dict(count=0, param=None, grad=None, exp_avg=None, exp_avg_sq=None)) == OK
    assert log_probs(one, log_probs=None) == OK                    # no output is wanted anywhere


@pytest.mark.parametrize("call", [log_probs, grad])
def test_logits(one, call):
    assert call(one, data_type=DT.FP64) == NOT_SUPPORT
    assert call(one, data_type=DT.FP8E4M3) == NOT_SUPPORT
    assert call(one, token_type=DT.UINT32) == NOT_SUPPORT
    assert call(one, logits=None) == PTR
    assert call(one, tokens=None) == PTR
    assert call(one, logits=A + 1) == PARA
    assert call(one, data_type=DT.FP32, logits=A + 2) == PARA
    assert call(one, tokens=A + 4) == PARA
    assert call(one, row_stride=7) == PARA
    assert call(one, row_stride=1 << 41) == PARA
    assert call(one, token_count=1 << 24) == PARA
    assert call(one, vocab_count=1 << 31, row_stride=1 << 31) == PARA
    assert call(one, vocab_start=(1 << 31) - 4) == PARA
    assert call(one, vocab_start=1 << 63) == PARA
    assert call(one, top_count=33) == PARA
    for scale in (0.0, -1.0, math.nan, math.inf, 1e-7, 2e6):
        assert call(one, scale=scale) == PARA, scale


def test_log_probs(one):
    assert log_probs(one, lse=A + 2) == PARA
    assert log_probs(one, top_count=2, top_ids=A + 4) == PARA
    assert log_probs(one, workspace=A + 8) == PARA
    assert log_probs(one, vocab_start=1) == PARA                    # the parts leave a gap
    assert log_probs(one, vocab_count=0, logits=None) == PARA       # no vocabulary at all
    assert log_probs(one, top_count=9) == PARA                      # more alternatives than entries
    need = model_ops.token_log_probs_workspace(1, 1 << 17, 20)
    assert need > 0
    for space, size in ((None, 0), (A, need - 1), (None, need)):
        assert log_probs(one, token_count=1, vocab_count=1 << 17, top_count=20, workspace=space, workspace_bytes=size) == MEMORY
    assert model_ops.token_log_probs_workspace(4096, 1 << 17, 20) == 0
    assert model_ops.token_log_probs_workspace(1, 1000, 20) == 0
    assert code(model_ops.token_log_probs_workspace, 1 << 24, 8, 0) == PARA
    assert code(model_ops.token_log_probs_workspace, 1, 1 << 31, 0) == PARA
    assert code(model_ops.token_log_probs_workspace, 1, 8, 33) == PARA
    assert model_ops.lib().HcclAmdTokenLogProbsWorkspace(1, 8, 0, None) == PTR
    assert model_ops.lib().HcclAmdTokenLogProbs(None, one, ctypes.c_void_p(STREAM)) == PTR
    assert model_ops.lib().HcclAmdTokenLogProbsGrad(None, one, ctypes.c_void_p(STREAM)) == PTR


def test_grad(one):
    assert grad(one, lse=None) == PTR
    assert grad(one, grad_logits=None) == PTR
    assert grad(one, grad_log_probs=None) == PTR                    # no gradient at all
    assert grad(one, grad_entropy=A) == PTR                         # without the entropy
    assert grad(one, top_count=2, grad_top_values=A) == PTR         # without the ids
    assert grad(one, grad_log_probs=None, top_count=0, grad_top_values=A, top_ids=A) == PTR
    assert grad(one, grad_row_stride=7) == PARA
    assert grad(one, grad_logits=0x90001) == PARA
    assert grad(one, lse=A + 1) == PARA
    assert grad(one, grad_log_probs=A + 2) == PARA
    # an overlap that is neither the logits themselves nor apart from them (rows of 8 bf16, 3 rows)
    assert grad(one, grad_logits=A + 2) == PARA
    assert grad(one, grad_logits=A + 16) == PARA
    assert grad(one, grad_logits=A, grad_row_stride=16) == PARA
    assert grad(one, row_stride=16, grad_row_stride=16, grad_logits=A + 14) == PARA


@pytest.mark.parametrize("which", ["tokens", "lse", "grad_log_probs", "entropy", "grad_entropy", "top_ids", "grad_top_values"])
def test_the_gradient_is_not_written_over_what_its_rows_are_computed_from(one, which):
    """Three rows of 8 floats, 20 floats apart, at D; every array but one lies elsewhere."""
    d = 0x90000
    entry = 8 if which in ("tokens", "top_ids") else 4
    size = 3 * entry * (2 if which.startswith(("top", "grad_top")) else 1)
    arrays = dict(tokens=A, lse=A, grad_log_probs=A, entropy=A, grad_entropy=A, top_ids=A, grad_top_values=A)
    row, stride, rows = 32, 80, 2 * 80 + 32
    for at in (d - size + entry, d, d + 24, d + stride, d + stride - entry, d + rows - entry):
        k = dict(arrays, **{which: at})
        assert grad(one, logits=A + 0x1000, grad_logits=d, grad_row_stride=20, top_count=2, **k) == PARA, (which, at - d)
    comms = hccl_amd.comm_init_all(2)      # a destroyed world refuses what passes the checks, before any launch
    hccl_amd.comm_destroy(comms[0])
    for at in (d - size, d + row, d + stride + row, d + stride - size, d + rows):
        if at % entry == 0:
            k = dict(arrays, **{which: at})
            assert grad(comms[1], logits=A + 0x1000, grad_logits=d, grad_row_stride=20, top_count=2, **k) == UNAVAIL, (which, at - d)
    # what is not read does not matter
    assert grad(comms[1], logits=A + 0x1000, grad_logits=d, tokens=d, grad_log_probs=None, entropy=A, grad_entropy=A) == UNAVAIL
    hccl_amd.comm_destroy(comms[1])


def test_norm(one):
    assert norm(one, result=None) == PTR
    assert norm(one, result=A + 2) == PARA
    assert norm(one, max_norm=math.nan) == PARA
    assert norm(one, max_norm=math.inf) == PARA
    assert norm(one, scale=math.inf) == PARA
    assert norm(one, workspace=A + 8) == PARA
    assert norm(one, [(None, 4, DT.FP32)]) == PTR
    assert norm(one, [(A, 4, DT.FP32), (A, 4, DT.INT32)]) == NOT_SUPPORT
    assert norm(one, [(A + 2, 4, DT.FP32)]) == PARA
    assert norm(one, [(A, 1 << 40, DT.FP32)]) == PARA
    assert norm(one, [(1 << 48, 4, DT.FP32)]) == PARA
    need = model_ops.grad_norm_workspace(1)
    assert norm(one, workspace=A, workspace_bytes=need - 1) == MEMORY
    assert model_ops.grad_norm_workspace(1000) > need
    assert code(model_ops.grad_norm_workspace, (1 << 40) + 1) == PARA
    assert model_ops.lib().HcclAmdGradNormWorkspace(1, None) == PTR
    assert model_ops.lib().HcclAmdGradNorm(None, 1, 1.0, 1.0, A, None, 0, one, ctypes.c_void_p(STREAM)) == PTR


def test_adamw(one):
    for field in ("param", "grad", "exp_avg", "exp_avg_sq"):
        assert adamw(one, {field: None}) == PTR, field
        assert adamw(one, {field: A + 2}) == PARA, field
    assert adamw(one, dict(master=A)) == NOT_SUPPORT                # beside 32-bit weights
    assert adamw(one, dict(param_type=DT.BFP16, grad_type=DT.FP16)) == NOT_SUPPORT
    assert adamw(one, dict(param_type=DT.FP64)) == NOT_SUPPORT
    assert adamw(one, dict(grad_type=DT.FP8E4M3)) == NOT_SUPPORT
    assert adamw(one, dict(count=1 << 40)) == PARA
    assert adamw(one, dict(param_type=DT.BFP16, grad_type=DT.BFP16, master=A + 2)) == PARA
    assert adamw(one, state_type=DT.FP8E4M3) == PTR                 # no scales
    assert adamw(one, dict(exp_avg_scale=A + 2, exp_avg_sq_scale=A), state_type=DT.FP8E4M3) == PARA
    assert adamw(one, state_type=DT.FP8E5M2) == NOT_SUPPORT
    assert adamw(one, step=0) == PARA
    for bad in (dict(lr=math.nan), dict(beta1=1.0), dict(beta1=-0.1), dict(beta2=1.0), dict(beta2=math.nan), dict(eps=-1.0),
                dict(eps=math.inf), dict(eps=1e-40), dict(eps=math.nan), dict(weight_decay=math.inf)):
        assert adamw(one, **bad) == PARA, bad
    assert adamw(one, step_on_device=A + 4) == PARA
    assert adamw(one, lr_on_device=A + 2) == PARA
    assert adamw(one, clip=A + 2) == PARA
    assert model_ops.lib().HcclAmdAdamW(None, 0, None, one, ctypes.c_void_p(STREAM)) == PTR
    with pytest.raises(TypeError):
        model_ops.adamw_tensors([dict(param=A, grad=A, exp_avg=A, exp_avg_sq=A, count=1, param_type=4, grad_type=4, step=1)])


def test_ranks_that_do_not_fit_together():
    """Every rank gets the same code, nothing is launched, and the next collective pairs up."""
    comms = hccl_amd.comm_init_all(2)

    def both(first, second):
        codes = [None, None]

        def call(r, k):
            codes[r] = log_probs(comms[r], **k)
        threads = [threading.Thread(target=call, args=(r, k)) for r, k in ((0, first), (1, second))]
        for t in threads:
            t.start()
        for t in threads:
            t.join(30)
        return codes
    whole = dict(vocab_start=0), dict(vocab_start=8)
    for change in (dict(token_count=4), dict(data_type=DT.FP16), dict(scale=2.0), dict(token_type=DT.INT32), dict(top_count=1),
                   dict(vocab_start=9), dict(vocab_start=0), dict(logits=None), dict(vocab_count=3, vocab_start=7)):
        got = both(whole[0], dict(whole[1], **change))
        assert got[0] == got[1] != OK, (change, got)
    try:
        # a norm against a log probability, and a norm with another scale
        codes = []
        hccl_amd.group_start()
        codes.append(norm(comms[0]))
        codes.append(log_probs(comms[1], vocab_start=8))
        assert code(hccl_amd.group_end) == PARA
        hccl_amd.group_start()
        codes.append(norm(comms[0], scale=1.0))
        codes.append(norm(comms[1], scale=2.0))
        assert code(hccl_amd.group_end) == PARA
        # a plain collective against one of these
        hccl_amd.group_start()
        codes.append(code(hccl_amd.all_reduce, comms[0], A, A, 1, DT.FP32, 0, STREAM))
        codes.append(norm(comms[1]))
        assert code(hccl_amd.group_end) == PARA
        # a rejected call settles its peer
        assert norm(comms[0], result=None) == PTR
        assert norm(comms[1]) == PTR
        # without outputs there is nothing to launch: both sides succeed, so the sequence is intact
        assert both(dict(log_probs=None), dict(log_probs=None, vocab_start=8)) == [OK, OK]
    finally:
        hccl_amd.comm_destroy(comms[0])
        assert log_probs(comms[1], vocab_start=8) == UNAVAIL
        assert grad(comms[1]) == UNAVAIL
        assert norm(comms[1]) == UNAVAIL
        assert adamw(comms[1]) == UNAVAIL
        hccl_amd.comm_destroy(comms[1])
    assert log_probs(comms[0]) == PARA                              # destroyed handles
    assert adamw(comms[1]) == PARA


def unfit_calls():
    """(operator, arguments) that no field of the C structures holds, or that are no numbers or buffers at all."""
    for k in (dict(token_count=-1), dict(token_count=1 << 64), dict(token_count=None), dict(vocab_count=-1),
              dict(vocab_start=-1), dict(row_stride=-1), dict(top_count=1 << 32), dict(top_count=-1), dict(scale=1e39),
              dict(scale="warm"), dict(data_type=1 << 40), dict(logits=-A), dict(logits=object()), dict(stream="x"),
              dict(workspace=A, workspace_bytes=-1), dict(workspace=A, workspace_bytes=1 << 64)):
        yield log_probs, k
    for k in (dict(tensors=[(A, -1, DT.FP32)]), dict(tensors=[(A, 4, 1 << 40)]), dict(tensors=[(A, 4)]),
              dict(tensors=[(object(), 4, DT.FP32)]), dict(max_norm=1e39), dict(max_norm=None), dict(scale="warm"),
              dict(result=object()), dict(stream="x"), dict(workspace=A, workspace_bytes=-1),
              dict(workspace=A, workspace_bytes=1 << 64)):
        yield norm, k


@pytest.mark.parametrize("call,bad", list(unfit_calls()))
@pytest.mark.parametrize("rank", [0, 1])
def test_a_call_whose_arguments_do_not_fit_releases_its_peers(call, bad, rank):
    """It raises, HcclError where it is a number that is out of range, its peer gets the same code at once, within a group or from
    a thread, and the collective that follows pairs up."""
    comms = hccl_amd.comm_init_all(2)
    try:
        for grouped in (False, True):
            got = {}

            def go(r, k):
                try:
                    got[r] = call(comms[r], **k)
                except Exception as e:
                    got[r] = e
            if grouped:
                hccl_amd.group_start()
                go(1 - rank, {})
                go(rank, bad)
                ended = code(hccl_amd.group_end)
                assert ended in (OK, PARA)
                assert got[1 - rank] == PARA or ended == PARA
            else:
                threads = [threading.Thread(target=go, args=(r, k), daemon=True) for r, k in ((rank, bad), (1 - rank, {}))]
                for t in threads:
                    t.start()
                for t in threads:
                    t.join(20)
                assert got.get(1 - rank) == PARA, got
            assert got[rank] == PARA or isinstance(got[rank], (TypeError, ValueError, ctypes.ArgumentError)), got
        # nothing to launch, but both ranks have to be at the same place of the sequence
        hccl_amd.group_start()
        assert log_probs(comms[0], log_probs=None, vocab_start=0) == OK
        assert log_probs(comms[1], log_probs=None, vocab_start=8) == OK
        assert code(hccl_amd.group_end) == OK
    finally:
        for c in comms:
            hccl_amd.comm_destroy(c)


def test_unfit_numbers_raise_the_library_s_error(one):
    """Not the packing's, and the local operators and the kept arrays too."""
    for call, bad in unfit_calls():
        if all(isinstance(v, (int, float)) for v in bad.values()):
            assert call(one, **bad) == PARA, bad
    assert log_probs(one, token_count=0, row_stride=-1) == PARA
    assert log_probs(one, data_type=DT.FP64) == NOT_SUPPORT
    for k in (dict(token_count=-1), dict(row_stride=-1), dict(grad_row_stride=1 << 64), dict(top_count=-1), dict(grad_logits=-A),
              dict(data_type=1 << 40)):
        assert grad(one, **k) == PARA, k
    for k in (dict(step=-1), dict(step=1 << 64), dict(clip=-A)):
        assert adamw(one, **k) == PARA, k
    assert adamw(one, dict(count=-1)) == PARA
    assert code(model_ops.adamw_tensors, [dict(param=A, grad=A, exp_avg=A, exp_avg_sq=A, count=-1, param_type=4, grad_type=4)]) == PARA
    assert code(model_ops.norm_tensors, [(A, -1, DT.FP32)]) == PARA
    # an array of the other operator's descriptors is none of this one's
    kept = model_ops.adamw_tensors([dict(param=A, grad=A, exp_avg=A, exp_avg_sq=A, count=1, param_type=4, grad_type=4)])
    with pytest.raises(TypeError):
        model_ops.grad_norm(one, kept, 1.0, A, stream=STREAM)


def test_a_broken_environment_fails_these_calls_too(monkeypatch):
    monkeypatch.setenv("HCCL_DETERMINISTIC", "perhaps")
    comms = hccl_amd.comm_init_all(1)
    try:
        for call in (log_probs, grad, norm, adamw):
            assert call(comms[0]) == PARA
    finally:
        hccl_amd.comm_destroy(comms[0])
