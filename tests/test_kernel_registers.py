"""Beside matrix instructions, vector registers are written by instructions that the compiler knows."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# (in the single-token attention, whose kernels have no matrix instruction)
APART = {"attn.hip": ["v_mov_b32 %0, 0"]}


def test_no_vector_instruction_is_inline_assembly():
    # A vector instruction that overwrites what a matrix instruction still reads, or is about to
    # write, needs wait states between.  The compiler puts them in front of its own instructions and of
    # none in an asm block, which it does not look into.
    found = 0
    for path in glob.glob(os.path.join(ROOT, "ai-research_amd", "csrc", "**", "*.h*"), recursive=True):
        text = re.sub(r"//[^\n]*", "", open(path).read())
        if "__builtin_amdgcn_mfma" not in text:
            continue
        for block in re.findall(r"\basm\b(?:\s+volatile)?\s*\((.*?)\)\s*;", text, flags=re.S):
            found += 1
            code = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', block.split(":")[0]))
            for instruction in re.split(r"\\n|;", code):
                name = instruction.replace("\\t", " ").strip()
                assert not name.startswith("v_") or name in APART.get(os.path.basename(path), []), (os.path.basename(path), name)
    assert found > 0
