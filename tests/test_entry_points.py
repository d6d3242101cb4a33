"""Declared argument types of kernel-library entry points against their C signatures (a wrong letter would shift every later argument)."""

import re
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1] / "lyra_b200"


def c_signature(name: str) -> str:
    for source in (ROOT / "csrc").rglob("*.cu"):
        found = re.search(r'extern "C" [\w ]+ ' + name + r"\(([^)]*)\)", source.read_text())
        if found:
            code = ""
            for arg in (a.strip() for a in found.group(1).split(",")):
                pointer = "*" in arg or arg.startswith("cudaStream_t")
                code += "p" if pointer else "l" if arg.startswith("long long") else "f" if arg.startswith("float") else "i"
            return code
    raise AssertionError(f"{name} is not defined in csrc")


def test_declared_argument_types_match_the_c_signatures():
    checked = 0
    for module in (ROOT / "ops").glob("*.py"):
        text = module.read_text()
        constants = dict(re.findall(r'^(_\w+_ARGS) = ("[pilf]+"(?: \+ "[pilf]+")*)$', text, re.M))
        for name, declared in re.findall(r'native\.function\("(\w+)", ((?:"[pilf]+"(?: \+ "[pilf]+")*)|_\w+)', text):
            declared = constants.get(declared, declared)
            assert "".join(re.findall(r'"([pilf]+)"', declared)) == c_signature(name), name
            checked += 1
    assert checked >= 6
