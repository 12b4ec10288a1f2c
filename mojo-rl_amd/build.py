"""Builds libmrl_hip.so for gfx950 with hipcc (cross-compiles without a GPU): one object per
translation unit, compiled side by side, then linked."""
import os
import re
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "libmrl_hip.so")
SOURCES = ["mrl_core.hip", "mrl_env.hip", "mrl_env_many.hip", "mrl_mlp.hip", "mrl_mlp3.hip", "mrl_fb.hip", "mrl_rows.hip", "mrl_ppo.hip", "mrl_policy.hip", "mrl_rollout.hip", "mrl_collect.hip", "mrl_update.hip", "mrl_shuffle.hip", "mrl_recurrence.hip", "mrl_muon.hip", "mrl_delta.hip", "mrl_delta_back.hip", "mrl_clip.hip", "mrl_glu.hip"]
# the 16-row collection kernels, a translation unit per hidden width
COLLECT16 = ["mrl_collect%s_h%d.hip" % (k, h) for k in ("16", "_walkers") for h in (256, 128, 64)]
SOURCES = COLLECT16 + SOURCES   # (the longest to compile go first)
# -ffp-contract=off: fp32/fp64 results follow the written order of operations (the GEMM inner
# loops spell out fmaf / MFMA themselves).  The -target-feature pair switches packed-fp32
# code generation off.
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-Wno-unused-value"]
# The collection kernels run a long env step inside a loop over the rollout steps.  The machine-level
# loop-invariant code motion lifts the double-precision constants of that step (the polynomial
# coefficients of exp / log / sincos, two registers each) out of the loop into registers of their own,
# the register allocator then spills them, and every use becomes a dependent load from private memory in
# the middle of the solver wavefront's chain.  Without that pass these kernels need no private memory.
# In the stand-alone env kernels the lifted constants push scalar registers out instead.  Where a saved scalar register is
# the first thing in a block, the register allocator of this compiler has been seen to put vector copies next, ahead of the
# instruction that widens the lane mask again, so that lanes outside the mask lose the value.  The flag makes that rarer, it
# does not rule it out: narrow_copies() looks for it in every unit.
EXTRA_FLAGS = {f: ["-mllvm", "-disable-machine-licm"] for f in ["mrl_collect.hip", "mrl_env.hip", "mrl_env_many.hip"] + COLLECT16}


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    out = "\n".join(l for l in proc.stdout.splitlines() if "packed-fp32-ops' is not a recognized feature" not in l)
    if proc.returncode != 0:
        raise RuntimeError("hipcc failed:\n" + out)
    if verbose and out.strip():
        print(out)


def build(verbose=False, incremental=False, jobs=8):
    """Compiles every translation unit (incremental=True: only those older than a source or header
    they could include) and links the library."""
    os.makedirs(OBJ, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hpp")]
    headers.append(os.path.join(HERE, "..", "include", "mrl.h"))
    newest_header = max(os.path.getmtime(h) for h in headers)
    todo, objs = [], []
    for s in SOURCES:
        src, obj = os.path.join(CSRC, s), os.path.join(OBJ, s[:-4] + ".o")
        objs.append(obj)
        fresh = os.path.exists(obj) and os.path.getmtime(obj) > max(os.path.getmtime(src), newest_header)
        if not (incremental and fresh):
            todo.append(["hipcc"] + FLAGS + EXTRA_FLAGS.get(s, []) + ["-c", src, "-o", obj])
    with ThreadPoolExecutor(max_workers=jobs) as pool:
        list(pool.map(lambda c: _run(c, verbose), todo))
    _run(["hipcc", "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs, verbose)
    return LIB


# ---- vector copies ahead of a widening lane mask
# A block where lanes join again opens with exec = exec | saved.  Behind register allocation, before blocks are merged,
# nothing may stand ahead of that but scalar instructions and scalar registers going to and from lanes of a vector register
# (which no mask holds back): a vector copy or a spill there leaves out the lanes that have not joined yet.
_WIDENS = re.compile(r"^\$exec = S_OR_B64(_term)? \$exec\b|= S_OR_SAVEEXEC_B64\b")
_OTHER_EXEC = re.compile(r"^\$exec = |\bimplicit-def (dead )?\$exec\b")
_HARMLESS = re.compile(r"= IMPLICIT_DEF\b|\b(V_READLANE_B32|V_WRITELANE_B32|SI_SPILL_S32_TO_VGPR|SI_RESTORE_S32_FROM_VGPR)\b")


def narrow_copies(lines):
    """(joins, faults) of a unit's machine code behind register allocation, the lines of it."""
    joins, faults, kernel, head, block = 0, [], None, None, None
    for line in lines:
        if line.startswith("name:"):
            kernel = line.split()[1]
        elif line.startswith("  bb."):
            block, head = line.split()[0], []
        elif head is not None and line.startswith("    ") and not line.startswith(("    liveins:", "    successors:")):
            ins = line.strip()
            if _WIDENS.search(ins):
                joins += 1
                faults += [(kernel, block, h) for h in head if re.search(r"\$[va]gpr\d", h) and not _HARMLESS.search(h)]
                head = None
            elif _OTHER_EXEC.search(ins):
                head = None
            else:
                head.append(ins)
    return joins, faults


def check_lane_masks(jobs=8):
    """Compiles every unit up to the end of register allocation; {unit: (joins, faults)}."""
    def one(unit):
        cmd = ["hipcc"] + FLAGS + EXTRA_FLAGS.get(unit, []) + ["--cuda-device-only", "-S", os.path.join(CSRC, unit), "-o", "-",
               "-mllvm", "-stop-after=virtregrewriter,2"]   # (scalar, whole-wavefront and vector registers: three passes)
        with subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.DEVNULL, text=True) as proc:
            found = narrow_copies(proc.stdout)
        if proc.returncode != 0:
            raise RuntimeError("hipcc failed: " + " ".join(cmd))
        return unit, found
    with ThreadPoolExecutor(max_workers=jobs) as pool:
        return dict(pool.map(one, SOURCES))


# ---- results of the matrix cores read too early
# A product's registers may be read some instructions behind it; the hardware does not wait for them, the compiler counts.  Behind
# a taken branch this compiler has been seen to count too few, down to one, and the reader took what had stood there before.
_STATES = (("16x16x32", 8), ("16x16x16", 8), ("16x16x4_f32", 10), ("32x32", 18))   # what it leaves within a block
_REGISTERS = re.compile(r"\b([va])\[(\d+):(\d+)\]|\b([va])(\d+)\b")
_WRITES_MEMORY = re.compile(r"^(ds_write|(global|buffer|flat|scratch)_(store|atomic))")


def _registers(text):
    found = set()
    for kind, first, last, other, alone in _REGISTERS.findall(text):
        found |= {other + alone} if alone else {kind + str(i) for i in range(int(first), int(last) + 1)}
    return found


def _kernels(lines):
    """{kernel: [(instruction, operands) or (label, None)]} of a unit's assembly, the lines of it."""
    kernels, code = {}, None
    for line in lines:
        label = re.match(r"^(\.LBB\d+_\d+|_Z\w+):", line)
        if label and label[1].startswith("_Z"):
            code = kernels.setdefault(label[1], [])
        elif label and code is not None:
            code.append((label[1], None))
        elif code is not None:
            op, _, rest = line.split(";")[0].strip().partition(" ")
            if op and not op.startswith("."):
                code.append((op, rest.strip()))
    return kernels


def early_reads(lines):
    """(products, faults) of a unit's assembly, the lines of it."""
    kernels, products, faults = _kernels(lines), 0, []
    for kernel, code in kernels.items():
        at = {op: i for i, (op, rest) in enumerate(code) if rest is None}
        for i, (op, rest) in enumerate(code):
            if rest is None or not op.startswith("v_mfma"):
                continue
            products += 1
            states = next((n for shape, n in _STATES if shape in op), 18)
            todo, seen = [(i + 1, 0, frozenset(_registers(rest.split(",")[0])))], set()
            while todo:
                j, waited, live = todo.pop()
                while j < len(code) and waited < states and live and (j, waited, live) not in seen:
                    seen.add((j, waited, live))
                    name, args = code[j]
                    j += 1
                    if args is None:
                        continue
                    waited += 1
                    if name == "s_nop":
                        waited += int(args)
                    elif name in ("s_endpgm", "s_setpc_b64"):
                        break
                    elif name == "s_branch":
                        j = at[args]
                    elif name.startswith("s_cbranch"):
                        todo.append((at[args], waited, live))
                    elif not name.startswith("s_"):
                        words = args.split(",")
                        written = set() if _WRITES_MEMORY.match(name) else _registers(words[0])
                        read = _registers(",".join(words[1:])) if written else _registers(args)
                        if name.startswith("v_mfma"):           # (the addend of a like product may follow at once)
                            read = _registers(",".join(words[1:3]))
                        elif written & live:                     # overwritten early: no better
                            read |= written
                        if read & live:
                            faults.append((kernel, op + " " + rest, name + " " + args, waited - 1))
                        live -= written | read
    return products, faults


def empty_masks(lines):
    """Kernels with a narrowed lane mask around nothing: what stood there, a copy of a register that the other way around has
    overwritten, has been seen to be lost."""
    kernel, last, found = None, "", []
    for line in lines:
        label = re.match(r"^(_Z\w+):", line)
        kernel = label[1] if label else kernel
        ins = line.split(";")[0].strip()
        if not ins or ins.startswith("."):
            continue
        saved = re.match(r"s_and_saveexec_b64 (s\[\d+:\d+\])", last)
        if saved and ins == "s_or_b64 exec, exec, " + saved[1]:
            found.append(kernel)
        last = ins
    return found


def stores_around_barriers(lines, name):
    """{kernel: stores to memory that a loop can come to again without a barrier} of the kernels that have `name` in theirs.  Where a loop
    hands LDS from one iteration to the next its wavefronts may be one barrier apart, and no more: every way around has one."""
    found = {}
    for kernel, code in _kernels(lines).items():
        if name not in kernel:
            continue
        at = {op: i for i, (op, rest) in enumerate(code) if rest is None}

        def behind(i):
            op, rest = code[i]
            if rest is None or not op.startswith("s_"):
                return [i + 1]
            if op in ("s_barrier", "s_endpgm", "s_setpc_b64"):
                return []
            if op == "s_branch":
                return [at[rest]]
            return [i + 1, at[rest]] if op.startswith("s_cbranch") else [i + 1]
        again = []
        for i, (op, rest) in enumerate(code):
            if rest is None or not op.startswith(("global_store", "buffer_store", "flat_store")):
                continue
            todo, seen = behind(i), set()
            while todo:
                j = todo.pop()
                if j < len(code) and j not in seen:
                    seen.add(j)
                    todo += behind(j)
            if i in seen:
                again.append(op + " " + rest)
        found[kernel] = again
    return found


def assembly(unit):
    """The lines of a unit's assembly."""
    cmd = ["hipcc"] + FLAGS + EXTRA_FLAGS.get(unit, []) + ["--cuda-device-only", "-S", os.path.join(CSRC, unit), "-o", "-"]
    proc = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.DEVNULL, text=True)
    if proc.returncode != 0:
        raise RuntimeError("hipcc failed: " + " ".join(cmd))
    return proc.stdout.splitlines()


def check_matrix_results(jobs=8):
    """Compiles every unit that uses the matrix cores to assembly; {unit: (products, faults, kernels with empty masks)}."""
    def one(unit):
        lines = assembly(unit)
        return unit, (*early_reads(lines), empty_masks(lines))
    units = []
    for unit in SOURCES:
        with open(os.path.join(CSRC, unit)) as f:
            if "mfma" in f.read():
                units.append(unit)
    with ThreadPoolExecutor(max_workers=jobs) as pool:
        return dict(pool.map(one, units))


if __name__ == "__main__":
    print(build(verbose=True, incremental="--incremental" in sys.argv))
    sys.exit(0)
