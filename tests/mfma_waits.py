"""Walks gfx950 assembly and lists the places where a matrix instruction's result is touched too soon.

The hardware does not hold back a vector instruction that reads or overwrites the result of a matrix
instruction still in flight: the compiler has to keep passes + 4 wait states between them (passes + 3 on the
parts before gfx950; 4 passes for 16x16x32 bf16, 8 for 32x32x16; every instruction counts for one, s_nop n
for n + 1).  hipcc has been seen to miss that across the end of a basic block, so this follows every path,
through branches.

  python mfma_waits.py FILE.s      exit status 1 if there is such a place"""
import re
import sys

PASSES = {"16x16x32": 4, "32x32x16": 8, "16x16x16": 4, "32x32x8": 8, "16x16x128": 8, "32x32x64": 16}
REG = re.compile(r"(?<![\w.])([va])(?:\[(\d+):(\d+)\]|(\d+))(?!\w)")


def registers(text):
    out = set()
    for kind, lo, hi, one in REG.findall(text):
        lo, hi = (int(one), int(one)) if one else (int(lo), int(hi))
        out.update((kind, i) for i in range(lo, hi + 1))
    return out


def functions(lines):
    name, body = None, []
    for line in lines:
        line = line.split(";")[0].rstrip()
        m = re.match(r"(\w+):", line)
        if m and not line.startswith(".L"):
            name, body = m.group(1), []
        elif line.startswith(".Lfunc_end"):
            if name and body:
                yield name, body
            name, body = None, []
        elif name is not None and (line.startswith(".LBB") or (line.startswith("\t") and not line.startswith("\t."))):
            body.append(line.strip())


def violations(body):
    code, label = [], {}
    for line in body:
        if line.startswith(".LBB"):
            label[line.split(":")[0]] = len(code)
        elif line:
            code.append(line)
    regs = [None] * len(code)

    def regs_of(i):
        if regs[i] is None:
            regs[i] = registers(code[i])
        return regs[i]

    def successors(i):
        op = code[i].split()[0]
        if op == "s_endpgm":
            return []
        if op == "s_branch":
            return [label[code[i].split()[1]]]
        nxt = [i + 1] if i + 1 < len(code) else []
        return nxt + ([label[code[i].split()[1]]] if op.startswith("s_cbranch") else [])

    bad = []
    for i, line in enumerate(code):
        if not line.startswith("v_mfma"):
            continue
        shape = re.search(r"_(\d+x\d+x\d+)_?", line).group(1)
        need = PASSES[shape] + 4
        dst = registers(line.split(None, 1)[1].split(",")[0])
        todo, seen = [(n, 0) for n in successors(i)], {}
        while todo:
            j, states = todo.pop()
            if states >= need or seen.get(j, need) <= states:
                continue
            seen[j] = states
            op = code[j].split()[0]
            if not op.startswith(("s_", "v_mfma")) and dst & regs_of(j):
                bad.append((i, line, states, code[j]))
                break
            width = int(code[j].split()[1]) + 1 if op == "s_nop" else 1
            if op.startswith("v_mfma") and dst <= registers(code[j].split(None, 1)[1].split(",")[0]):
                continue  # a later matrix instruction takes the result over
            todo += [(n, states + width) for n in successors(j)]
    return bad


def audit(path):
    found = {}
    for name, body in functions(open(path)):
        if any(line.startswith("v_mfma") for line in body):
            found[name] = violations(body)
    return found


if __name__ == "__main__":
    total = 0
    for name, bad in audit(sys.argv[1]).items():
        print(name[:100], len(bad))
        for b in bad[:3]:
            print("   ", b)
        total += len(bad)
    sys.exit(1 if total else 0)
