"""Builds the CPU emulation of libhccl_amd_model_ops.so for the tests: test infrastructure only, never loaded by the package.

    build/libhccl_amd_model_ops_emu_asan.so   entry points and kernels of hccl_amd/csrc/model_ops on top of
                                              build/libhccl_amd_emu_asan.so, run by lanes/lanes.cc

The sources are compiled as they are, against the stand-in HIP header of lanes/, but for the two things below."""
import hashlib
import os
import shutil
import subprocess

import build_emu

HERE = build_emu.HERE
CSRC = os.path.join(build_emu.CSRC, "model_ops")
SRC = os.path.join(build_emu.BUILD, "src_model_ops")
LANES = os.path.join(HERE, "lanes")
LIB = os.path.join(build_emu.BUILD, "libhccl_amd_model_ops_emu_asan.so")
BUILTINS = {"readfirstlane": "ReadFirstLane", "readlane": "ReadLane", "update_dpp": "UpdateDpp", "exp2f": None, "sqrtf": None,
            "permlane16_swap": "Permlane16Swap", "permlane32_swap": "Permlane32Swap", "cvt_f32_fp8": "WidenFp8",
            "cvt_pk_fp8_f32": "NarrowFp8Pair", "rcpf": "Reciprocal"}
# an empty statement that keeps a value in a register, and dynamic LDS
RULES = [('asm("" : "+v"(w[s][i]));', ""),
         ("extern __shared__ uint16_t groupMost[];", "uint16_t* const groupMost = static_cast<uint16_t*>(lanes::DynamicLds());")]


def sources():
    """name -> text of the sources as they are compiled."""
    texts = {}
    for fn in sorted(os.listdir(CSRC)):
        if fn.endswith((".h", ".hip", ".cc")):
            text = open(os.path.join(CSRC, fn)).read()
            for old, new in RULES:
                text = text.replace(old, new)
            code = "\n".join(line.split("//")[0] for line in text.split("\n"))
            assert "asm" not in code and "extern __shared__" not in code, "%s: no rule for this in build_model_ops.py" % fn
            texts[fn[:-4] + ".cc" if fn.endswith(".hip") else fn] = text
    return texts


def build():
    """Returns the paths of the two emulation libraries (built if their sources changed)."""
    base = build_emu.build(asan=True)
    texts = sources()
    stamp = hashlib.sha256(repr((sorted(texts.items()), open(base + ".stamp").read())).encode())
    for fn in (os.path.join(LANES, "lanes.cc"), os.path.join(LANES, "hip", "hip_runtime.h"), os.path.abspath(__file__)):
        stamp.update(open(fn, "rb").read())
    if os.path.exists(LIB) and os.path.exists(LIB + ".stamp") and open(LIB + ".stamp").read() == stamp.hexdigest():
        return base, LIB
    shutil.rmtree(SRC, ignore_errors=True)
    os.makedirs(SRC)
    for fn, text in texts.items():
        open(os.path.join(SRC, fn), "w").write(text.replace('"../host.h"', '"host.h"'))
    flags = [build_emu.CLANG, "-x", "c++", "-std=c++17", "-O1", "-gline-tables-only", "-fPIC", "-ffp-contract=off", "-mf16c",
             "-mfma", "-pthread", "-Wno-unknown-attributes", "-Wno-ignored-attributes", "-I" + LANES,
             "-I" + os.path.join(build_emu.ROOT, "include"), "-I" + SRC, "-I" + build_emu.SRC, "-Daddress_space(x)="]
    flags += ["-D__builtin_amdgcn_%s=%s" % (k, "lanes::" + v if v else k) for k, v in BUILTINS.items()]
    flags += build_emu.SANITIZE["asan"]
    jobs = []
    for unit in [os.path.join(SRC, fn) for fn in texts if fn.endswith(".cc")] + [os.path.join(LANES, "lanes.cc")]:
        obj = os.path.join(SRC, os.path.basename(unit)[:-3] + ".o")
        jobs.append((obj, unit, subprocess.Popen(flags + ["-c", unit, "-o", obj], stderr=subprocess.PIPE)))
    for _, unit, proc in jobs:
        build_emu._reap((unit, proc))
    subprocess.check_call([build_emu.CLANG, "-shared", "-pthread", "-o", LIB] + [obj for obj, _, _ in jobs] +
                          [base, "-Wl,-rpath," + build_emu.BUILD, "-fsanitize=address", "-shared-libsan"])
    open(LIB + ".stamp", "w").write(stamp.hexdigest())
    return base, LIB


if __name__ == "__main__":
    print(build()[1])
