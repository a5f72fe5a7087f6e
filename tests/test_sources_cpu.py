"""What the kernels' sources have to state, since a build that happens to be right does not show that it is missing."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "krikil_rs_b200", "csrc")
# instructions that read, write or order memory
MEMORY = re.compile(r"\b(cp\.async|mbarrier|fence|membar|barrier|ldmatrix|stmatrix|ld\.|st\.|red\.|atom\.|griddepcontrol|"
                    r"cluster\.sync)")


def assembly(text):
    """(line, statement) of each asm statement."""
    for m in re.finditer(r"\basm\b[^(;]*\(", text):
        end, depth, quoted = m.end(), 1, False
        while depth:
            c = text[end]
            if c == '"' and text[end - 1] != "\\":
                quoted = not quoted
            elif not quoted:
                depth += (c == "(") - (c == ")")
            end += 1
        yield text.count("\n", 0, m.start()) + 1, text[m.start():end]


def test_assembly_that_touches_or_orders_memory_says_so():
    """Else the compiler may move loads and stores across it: those of a copy's target to before the wait for the copy."""
    seen, bad = 0, []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        with open(path) as f:
            for line, statement in assembly(f.read()):
                if MEMORY.search(statement):
                    seen += 1
                    if "volatile" not in statement or '"memory"' not in statement:
                        bad.append(f"{os.path.basename(path)}:{line}")
    assert seen > 10 and not bad, bad
