"""CPU tier: what the compiler made of the model operators' kernels, read from the built library's own code objects, as
test_kernel_resources.py does for the data plane's."""
import os
import re
import subprocess

import pytest

from hccl_amd import model_ops

LLVM = "/opt/rocm/llvm/bin"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


@pytest.fixture(scope="module")
def objects(tmp_path_factory):
    """One code object per translation unit."""
    if not os.path.exists(model_ops.LIB_PATH):
        pytest.fail("%s is missing: build the library first" % model_ops.LIB_PATH)
    tmp = tmp_path_factory.mktemp("model_ops")
    fat = tmp / "fat.bin"
    subprocess.check_call([LLVM + "/llvm-objcopy", "--dump-section", ".hip_fatbin=%s" % fat, model_ops.LIB_PATH,
                           str(tmp / "unused.so")])
    data = fat.read_bytes()
    starts = [m.start() for m in re.finditer(re.escape(MAGIC), data)]
    found = []
    for i, at in enumerate(starts):
        bundle, obj = tmp / ("bundle%d.bin" % i), tmp / ("code%d.o" % i)
        bundle.write_bytes(data[at:starts[i + 1] if i + 1 < len(starts) else len(data)])
        subprocess.check_call([LLVM + "/clang-offload-bundler", "--unbundle", "--type=o",
                               "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", "--input=%s" % bundle, "--output=%s" % obj])
        found.append(obj)
    return found


@pytest.fixture(scope="module")
def kernels(objects):
    found = []
    for obj in objects:
        notes = subprocess.run([LLVM + "/llvm-readelf", "--notes", str(obj)], stdout=subprocess.PIPE, text=True,
                               check=True).stdout
        for block in re.split(r"\n\s+- \.agpr_count:", notes)[1:]:
            def field(key, block=block):
                return re.search(r"\.%s:\s+(\S+)" % key, block).group(1)
            found.append({"name": field("name"), "vgpr": int(field("vgpr_count")), "spills": int(field("vgpr_spill_count")),
                          "private": int(field("private_segment_fixed_size")), "args": int(field("kernarg_segment_size")),
                          "lds": int(field("group_segment_fixed_size"))})
    return found


def test_every_kernel_is_there(kernels):
    count = lambda part: sum(part in k["name"] for k in kernels)  # noqa: E731
    assert count("LogProbsKernel") == 18         # three types, three workgroup sizes, with and without alternatives
    assert count("LogProbsJoinKernel") == 3
    assert count("LogProbsGradKernel") == 6      # three types, with and without alternatives
    assert count("NormBatchKernel") == count("NormJoinKernel") == 1
    assert count("AdamWKernel") == 22            # eleven combinations of types, two kinds of states
    assert len(kernels) == 18 + 3 + 6 + 2 + 22


def test_no_kernel_spills_vectors_or_uses_private_memory(kernels):
    bad = [k for k in kernels if k["spills"] or k["private"]]
    assert not bad, bad


def test_registers_leave_room_for_the_wavefronts_the_forms_count_on(kernels):
    """512 registers per SIMD: eight wavefronts up to 64, seven up to 72; a workgroup of 1024 threads has a CU to itself."""
    for k in kernels:
        if "LogProbsKernel" in k["name"]:
            limit = 128 if "j1024" in k["name"] else 72 if "Lb1E" in k["name"] else 64
        else:
            limit = 72
        assert k["vgpr"] <= limit, k
        assert k["args"] <= 4096, k
        assert k["lds"] <= 20 * 1024, k


def test_no_packed_32_bit_arithmetic(objects):
    """Two-at-a-time 32-bit multiplies and adds are switched off for the whole build."""
    for obj in objects:
        text = subprocess.run([LLVM + "/llvm-objdump", "-d", "--mcpu=gfx950", str(obj)], stdout=subprocess.PIPE, text=True,
                              check=True).stdout
        assert "s_endpgm" in text
        assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text), obj
