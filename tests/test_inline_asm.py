"""Inline assembly of the kernels names every register that it writes by itself."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "mini-megatron_amd", "mi_adamw", "csrc")
REGISTER = re.compile(r"\b(m0|vcc|exec|scc|s\d+|v\d+)\b")


def statements():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.hip")) +
                       glob.glob(os.path.join(CSRC, "*.h"))):
        text = open(path).read()
        for found in re.finditer(r"\basm(?:\s+volatile)?\s*\(", text):
            depth, at = 1, found.end()
            while depth:
                depth += {"(": 1, ")": -1}.get(text[at], 0)
                at += 1
            yield os.path.basename(path), text[found.end():at - 1]


def test_written_registers_are_clobbered():
    seen = 0
    for name, body in statements():
        code, *operands = re.split(r'(?<=")\s*:', body, maxsplit=1)
        lines = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', code)).split("\\n\\t")
        clobbers = re.findall(r'"([^"]*)"', body.rsplit(":", 1)[1]) if operands else []
        for line in lines:
            words = line.split(None, 1)
            first = words[1].split(",")[0] if len(words) > 1 else ""
            for register in REGISTER.findall(first):
                seen += 1
                assert register in clobbers, f"{name}: {line} without a clobber of {register}"
    assert seen
