"""The training operators' product kernels as they were built (no GPU needed): their matrix instructions are asm statements whose accumulators stay in
their registers (ccsm_train_ops_mfma.h), so hipcc pads none of their hazards.  Read from the gfx950 code objects inside libccsm_train.so and
checked by the rules of tools/isa_gate.py: every accumulator tied, two states between a vector write and the product that reads it, seven
between a product and whatever else touches its result, along the code and around each loop; no scratch."""
import os
import re
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tools"))
LIB = os.path.join(ROOT, "ccsmeth_amd", "lib", "libccsm_train.so")
LLVM = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "lib", "llvm", "bin")
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"

pytestmark = pytest.mark.skipif(not os.path.exists(LIB) or not os.path.exists(os.path.join(LLVM, "llvm-objdump")), reason="libccsm_train.so or llvm-objdump is missing")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{name: (instructions, their addresses, {index of a branch: address it goes to}, scratch bytes, spilled registers)} of the product kernels"""
    d = str(tmp_path_factory.mktemp("co"))
    fat = os.path.join(d, "fat.bin")
    subprocess.run([os.path.join(LLVM, "llvm-objcopy"), "--dump-section", ".hip_fatbin=" + fat, LIB, os.path.join(d, "unused.so")], check=True)
    data = open(fat, "rb").read()
    at = [m.start() for m in re.finditer(MAGIC, data)] + [len(data)]
    out = {}
    for k in range(len(at) - 1):                                   # one bundle for each object file
        part, co = os.path.join(d, "part%d" % k), os.path.join(d, "dev%d.co" % k)
        open(part, "wb").write(data[at[k]:at[k + 1]])
        subprocess.run([os.path.join(LLVM, "clang-offload-bundler"), "--unbundle", "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", "--input=" + part, "--output=" + co],
                       check=True)
        notes = subprocess.run([os.path.join(LLVM, "llvm-readelf"), "--notes", co], check=True, capture_output=True, text=True).stdout
        meta = {}
        for entry in notes.split("  - .agpr_count")[1:]:
            f = dict(re.findall(r"^    \.(\w+):\s+(\S+)", entry, re.M))
            meta[f["name"]] = (int(f["private_segment_fixed_size"]), int(f["vgpr_spill_count"]))
        names = [n for n in meta if re.search(r"product_(pair_)?kernelIDF16", n)]                       # of 16-bit types
        if not names:
            continue
        text = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", "--no-show-raw-insn", "--disassemble-symbols=" + ",".join(names), co], check=True, capture_output=True,
                              text=True).stdout
        for m in re.finditer(r"^([0-9a-f]+) <(\S+)>:\n((?:[ \t].*\n)+)", text, re.M):
            base, name = int(m.group(1), 16), m.group(2)
            ins, where, goes = [], [], {}
            for ln in m.group(3).splitlines():
                p = re.match(r"\s+(\S.*?)\s*// ([0-9A-F]+):(.*)$", ln)
                if not p:
                    continue
                to = re.search(r"<\S+?\+0x([0-9a-f]+)>", p.group(3))
                if p.group(1).startswith(("s_cbranch", "s_branch")) and to:
                    goes[len(ins)] = base + int(to.group(1), 16)
                ins.append(p.group(1))
                where.append(int(p.group(2), 16))
            out[name] = (ins, where, goes) + meta[name]
    return out


def findings(ins, where, goes, report):
    import isa_gate
    bad, products, tied = isa_gate.check_hazards("straight", ins, report)
    loops = 0
    for i, to in goes.items():
        if to in where and where.index(to) <= i and any(x.startswith("v_mfma") for x in ins[where.index(to):i]):
            body = ins[where.index(to):i + 1]
            bad += isa_gate.check_hazards("loop", body + body, report)[0]
            loops += 1
    return bad, products, tied, loops


def test_product_kernels(kernels):
    assert len(kernels) == 16, sorted(kernels)                     # two types, two tiles, three forms of the operands and the pair of two
    for name, (ins, where, goes, scratch, spilled) in kernels.items():
        said = []
        bad, products, tied, loops = findings(ins, where, goes, said.append)
        assert bad == 0, "\n".join(said)
        assert products and tied == products and loops >= (2 if "pair" in name else 1), (name, products, tied, loops)
        assert scratch == 0 and spilled == 0, (name, scratch, spilled)


def test_the_check_sees_a_missing_wait(kernels):
    """the same instructions without those between the last product and the first reader of its result"""
    import isa_gate
    ins, where, _, _, _ = next(iter(kernels.values()))
    last = max(k for k, x in enumerate(ins) if x.startswith("v_mfma"))
    result = isa_gate.regs(isa_gate.operands(ins[last])[0])
    reader = next(k for k in range(last + 1, len(ins)) if isa_gate.all_vregs(isa_gate.operands(ins[k])) & result)
    assert findings(ins[:last + 1] + ins[reader:], where, {}, lambda s: None)[0] > 0
    assert findings(ins[:last + 1] + ["s_nop 6"] + ins[reader:], where, {}, lambda s: None)[0] < findings(ins[:last + 1] + ins[reader:], where, {}, lambda s: None)[0]
