"""Kernels that write matrix instructions out themselves: the compiler does not see that their sums come late.  In the compiled program of every such kernel
what is read of the sums comes out of the wait (an asm statement behind the wait's that takes every sum and gives it back), never out of the product, so that no
reading can be moved before the wait."""
import re
import subprocess

import pytest

from spyinfer_amd.kernels import build

#: what hands a value on without reading it
MOVES = ("phi", "extractvalue", "freeze", "bitcast")


def compiled(source, tmp_path, *options):
    out = str(tmp_path / "program")
    done = subprocess.run([build._hipcc()] + build.HIPCC_FLAGS + ["-I", build.CSRC, "-S", *options, "--cuda-device-only", build.CSRC + "/" + source + ".hip", "-o", out],
                          stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    assert done.returncode == 0, done.stdout.decode(errors="replace")
    with open(out) as f:
        return f.read()


def functions(source, tmp_path):
    return re.findall(r"^define [^\n]*?@(\S+?)\([^\n]*\{\n(.*?)^\}", compiled(source, tmp_path, "-emit-llvm"), re.S | re.M)


def sums_read_early(body):
    """(products, sums that the wait gives back, instructions that read a sum which comes from a product past no wait)."""
    lines = [x.strip() for x in body.split("\n")]
    made = dict((m.group(1), m.group(2)) for m in (re.match(r"(%[\w.]+) = (.*)", x) for x in lines) if m)
    is_product = lambda x: " asm " in x and "v_mfma" in x
    is_wait = lambda x: " asm " in x and re.search(r'asm sideeffect "", "=a', x) is not None
    late = {n for n, x in made.items() if is_product(x)}
    while True:              # (a sum handed on is a sum)
        more = {n for n, x in made.items() if n not in late and x.startswith(MOVES) and late & set(re.findall(r"%[\w.]+", x))}
        if not more:
            break
        late |= more
    early = [x for x in lines if late & set(re.findall(r"%[\w.]+", x.split(" = ", 1)[-1]))
             and not (is_product(x) or is_wait(x) or x.split(" = ", 1)[-1].startswith(MOVES))]
    return sum(map(is_product, lines)), sum(map(is_wait, lines)), early


@pytest.mark.parametrize("source,kernels", [("gemm_q8", 13), ("gemm_q8_tall", 15), ("gemm_rows_tall", 24)])
def test_sums_are_read_behind_the_wait(source, kernels, tmp_path):
    found = 0
    for name, body in functions(source, tmp_path):
        products, waits, early = sums_read_early(body)
        if products:
            found += 1
            assert waits > 0 and not early, (name, waits, early[:3])
            # the wait itself stands between the last product and the first sum that it gives back
            asm = [x for x in body.split("\n") if " asm sideeffect " in x]
            last, first = max(i for i, x in enumerate(asm) if "v_mfma" in x), min(i for i, x in enumerate(asm) if '"", "=a' in x)
            assert any("s_nop 15" in x for x in asm[last:first]), name
    assert found == kernels


def test_held_blocks_listing(tmp_path):
    """The blocks of gemm_q8.hip that write their products out, as machine code: two wait states before a product's operands may have been written by an ordinary
    instruction, and the sums' registers read only behind the two long waits."""
    found = 0
    for name, body in re.findall(r"^(_Z\d+gemm_q8_kernel\S*):(.*?)^\.Lfunc_end", compiled("gemm_q8", tmp_path), re.S | re.M):
        written = [x.strip() for part in re.findall(r"#ASMSTART(.*?)#ASMEND", body, re.S) for x in part.split("\n")]
        if not any(x.startswith("v_mfma") for x in written):
            continue
        found += 1
        lines = [x.split(";")[0].strip() for x in body.split("\n")]
        lines = [x for x in lines if x and not x.startswith(".")]
        assert sum(x.startswith("v_mfma") for x in lines) == sum(x.startswith("v_mfma") for x in written)         # (all of a kernel's or none)
        settled, read = True, 0
        for i, x in enumerate(lines):
            if x.startswith("v_mfma"):
                settled = False
                assert lines[i - 1] == "s_nop 1" or (lines[i - 1].startswith("v_mfma") and lines[i - 2] == "s_nop 1"), (name, lines[i - 2:i + 1])
            elif (x == "s_nop 15" and lines[i - 1] == "s_nop 15") or x.startswith(("s_branch", "s_endpgm")):
                settled = True
            elif x.startswith("v_accvgpr_read") or (re.match(r"(ds_write|ds_store|global_store|buffer_store|scratch_store|v_)", x) and re.search(r"\ba(\d|\[)", x.split(",", 1)[-1])):
                read += 1
                assert settled, (name, lines[i - 2:i + 1])
        assert read > 0, name
    assert found == 13


def test_the_look_finds_an_early_reading():
    product = '%1 = tail call { <4 x i32>, <4 x i32> } asm sideeffect "v_mfma_i32 $0, $2, $4, $0", "=a,=a,v,v,v,0,1"(...)\n%2 = extractvalue { <4 x i32>, <4 x i32> } %1, 0\n'
    wait = '%3 = tail call <4 x i32> asm sideeffect "", "=a,0"(<4 x i32> %2)\n'
    assert sums_read_early(product + wait + "store <4 x i32> %3, ptr %p")[2] == []
    assert sums_read_early(product + wait + "store <4 x i32> %2, ptr %p")[2] == ["store <4 x i32> %2, ptr %p"]
    assert sums_read_early(product + wait + "%4 = phi <4 x i32> [ %2, %a ], [ %9, %b ]\n%5 = extractelement <4 x i32> %4, i64 0")[2] == ["%5 = extractelement <4 x i32> %4, i64 0"]
