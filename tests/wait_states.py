"""Matrix products whose result is used too soon, in the assembly of this library's
own kernels.

Nothing in the hardware holds an instruction back until a matrix product before it
has written its result: the compiler puts wait states between them.  It counts
them within a block and over most branches, but not over every one (a product, a
branch over a block that is rarely taken, and the result's first use behind it:
the use read the registers' old values).  `early_uses` follows every way out of
every product."""
import re

# wait states that the compiler leaves between a product and a vector
# instruction that reads or overwrites its result
STATES = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x32_f16": 8,
          "v_mfma_i32_16x16x64_i8": 8, "v_mfma_f32_16x16x4_f32": 10}
MEMORY = ("ds_", "global_", "buffer_", "flat_", "scratch_")


def _registers(operand):
    m = re.match(r"-?\|?([va])\[(\d+):(\d+)\]", operand)
    if m:
        return {(m[1], i) for i in range(int(m[2]), int(m[3]) + 1)}
    m = re.match(r"-?\|?([va])(\d+)\b", operand)
    return {(m[1], int(m[2]))} if m else set()


def _of(operands):
    return set().union(set(), *map(_registers, operands))


def functions(text):
    """{name: [(opcode, operands, line)]} of an assembly file; labels are entries
    with the opcode 'label'."""
    out, body = {}, None
    for line in text.splitlines():
        m = re.match(r"(_Z\w+):", line)
        if m:
            body = out.setdefault(m[1], [])
            continue
        if line.startswith(".Lfunc_end"):
            body = None
        if body is None:
            continue
        m = re.match(r"(\.LBB\w+):", line)
        if m:
            body.append(("label", [m[1]], line))
            continue
        code = line.split(";")[0].strip()
        if not code or code.startswith("."):
            continue
        op, _, rest = code.partition("\t") if "\t" in code else code.partition(" ")
        operands = [a.strip() for a in re.split(r",(?![^\[]*\])", rest)] if rest.strip() else []
        body.append((op, operands, code))
    return out


def _uses(op, operands, line):
    """(registers read, registers written) of an instruction that is no product."""
    if op.startswith("v_cmp") or op.startswith("ds_write") or "_store" in op or \
            ("atomic" in op and "sc0" not in line) or op.startswith("v_readfirstlane"):
        return _of(operands), set()
    return _of(operands[1:]), _of(operands[:1])


def early_uses(text):
    """(number of products, ["function: product | use"]) of an assembly file."""
    found, products = [], 0
    for name, body in functions(text).items():
        labels = {b[1][0]: i for i, b in enumerate(body) if b[0] == "label"}
        for i, (op, operands, line) in enumerate(body):
            if not op.startswith("v_mfma"):
                continue
            products += 1
            result, need = _registers(operands[0]), STATES[op]
            best, todo = {}, [(i + 1, 0)]
            while todo:
                j, passed = todo.pop()
                while j < len(body) and passed < need and best.get(j, need) > passed:
                    best[j] = passed
                    o, args, code = body[j]
                    j += 1
                    if o == "label":
                        continue
                    if o == "s_endpgm":
                        break
                    if o.startswith("v_mfma"):
                        if _of(args[1:3]) & result:
                            found.append(f"{name}: {line} | {code}")
                        if _registers(args[0]) & result:
                            break               # the chain's next product: its own result
                    elif o.startswith(("v_",) + MEMORY):
                        read, written = _uses(o, args, code)
                        if read & result or (o.startswith("v_") and written & result):
                            found.append(f"{name}: {line} | {code}")
                            break
                        if written & result:
                            break               # a load, long after
                    passed += int(args[0], 0) + 1 if o == "s_nop" else 1
                    if o == "s_branch":
                        j = labels[args[0]]
                    elif o.startswith("s_cbranch"):
                        todo.append((labels[args[0]], passed))
    return products, found
