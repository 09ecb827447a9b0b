"""Checks, in the built code, that no kernel touches the result of an LDS read before it has waited for it, and that matrix
instructions written as assembly have the distances that they need.

usage: lds_reads.py [path/to/libldm_hip.so] [kernel name regex]      exit status 1 when a kernel breaks one of the rules

The matrix kernels of linear.hip read their fragments by inline assembly and wait for them later: the compiler takes such a
register as written at once, so a copy, a spill or another value in it between the read and the wait would be wrong without any
error.  This walks every kernel's control flow graph.  LDS operations of a wave end in order, so a read is complete behind a wait
for lgkmcnt(n) if at least n LDS operations were issued after it on every way there; until then no instruction may name a
register that it writes.

The matrix instructions of the 256 tile (ASM_MFMA) are inline assembly too, so the compiler inserts no wait states around them:
  a vector instruction writes a register -> a matrix instruction reads it: two wait states between;
  a matrix instruction (of up to eight passes) writes -> anything but the accumulation into the same registers touches it: 11.
An instruction is one wait state, s_nop n is n + 1, and a matrix instruction four: the next one cannot start earlier."""
import os
import re
import subprocess
import sys
import tempfile

if __package__ in (None, ""):
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from tools.kernel_resources import LLVM, MAGIC  # noqa: E402

LINE = re.compile(r"^\s+(\S+)\s*(.*?)\s*// ([0-9A-F]{12}):")
REG = re.compile(r"\b([va])(?:(\d+)\b|\[(\d+):(\d+)\])")
ASM_MFMA = re.compile(r"gemm_kernelI\S*Li8E")            # kernels whose matrix instructions are inline assembly
FAR = 16                                               # lgkmcnt waits for at most 15


def code_objects(lib, tmp):
    """The gfx950 code objects inside `lib`, as files."""
    fat = os.path.join(tmp, "fat.bin")
    subprocess.run(["objcopy", "-O", "binary", "--only-section=.hip_fatbin", lib, fat], check=True)
    with open(fat, "rb") as fh:
        blob = fh.read()
    starts = [m.start() for m in re.finditer(re.escape(MAGIC), blob)]
    for i, st in enumerate(starts):
        part, co = os.path.join(tmp, f"bundle{i}.bin"), os.path.join(tmp, f"dev{i}.co")
        with open(part, "wb") as fh:
            fh.write(blob[st: starts[i + 1] if i + 1 < len(starts) else len(blob)])
        r = subprocess.run([f"{LLVM}/clang-offload-bundler", "--unbundle", "--type=o", f"--input={part}",
                            "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", f"--output={co}"], capture_output=True, text=True)
        if r.returncode == 0 and os.path.exists(co) and os.path.getsize(co):
            yield co


def functions(listing):
    """{name: [(address, mnemonic, operands)]} of a disassembly."""
    out, cur = {}, None
    for line in listing.splitlines():
        m = re.match(r"^[0-9a-f]{16} <(.+)>:$", line)
        if m:
            cur = out.setdefault(m.group(1), [])
            continue
        m = LINE.match(line)
        if m and cur is not None:
            cur.append((int(m.group(3), 16), m.group(1), m.group(2)))
    return out


def regs(operands):
    s = set()
    for m in REG.finditer(operands):
        lo = int(m.group(2) or m.group(3))
        s.update((m.group(1), r) for r in range(lo, int(m.group(4) or lo) + 1))
    return s


def successors(code):
    """For each instruction the ones that may follow it."""
    at = {a: i for i, (a, _, _) in enumerate(code)}
    n, succ = len(code), []
    for i, (addr, op, args) in enumerate(code):
        nxt = [i + 1] if i + 1 < n else []
        if op.startswith(("s_branch", "s_cbranch")):
            off = int(args.split()[-1], 0) & 0xFFFF
            target = at[addr + 4 + 4 * (off - 0x10000 if off & 0x8000 else off)]
            nxt = [target] if op.startswith("s_branch") else nxt + [target]
        elif op == "s_endpgm":
            nxt = []
        elif op.startswith(("s_setpc", "s_swappc", "s_call", "s_subvector")):
            raise ValueError(f"{op} at {addr:x}: not followed")
        succ.append(nxt)
    return succ


def check(code):
    """Touches of unfinished reads [(address, instruction, registers)] of one kernel, and how many LDS reads it has."""
    succ, info = successors(code), []
    n, reads = len(code), 0
    for addr, op, args in code:
        lds = op.startswith("ds_") and not op.startswith("ds_nop")
        dst = set()
        if lds and re.match(r"ds_(read|load|bpermute|permute|swizzle|consume|append|.*_rtn)", op):
            dst = regs(args.split(",")[0])
            reads += 1
        m = re.search(r"lgkmcnt\((\d+)\)", args) if op == "s_waitcnt" else None
        info.append((lds, dst, regs(args), int(m.group(1)) if m else None))
    # state in front of an instruction: register -> the least number of LDS operations issued after its read
    state = [None] * n
    state[0] = {}
    work, bad = [0], {}
    while work:
        i = work.pop()
        cur = state[i]
        lds, dst, named, wait = info[i]
        if wait is not None:
            cur = {r: k for r, k in cur.items() if k < wait}
        hit = named & cur.keys()
        if hit:
            bad[i] = hit
        if lds:
            cur = {r: min(k + 1, FAR) for r, k in cur.items()}
            cur.update((r, 0) for r in dst)
        for j in succ[i]:
            old = state[j]
            if old is None:
                state[j] = cur
                work.append(j)
                continue
            new = dict(old)
            for r, k in cur.items():
                new[r] = min(k, new.get(r, k))
            if new != old:
                state[j] = new
                work.append(j)
    return [(code[i][0], " ".join(code[i][1:]), sorted(r)) for i, r in sorted(bad.items())], reads


def _flow(n, succ, first, step):
    """States {register: wait states since it was written} in front of every instruction, least over all ways."""
    state = [None] * n
    state[0], work = first, [0]
    while work:
        i = work.pop()
        cur = step(i, state[i])
        for j in succ[i]:
            old = state[j]
            new = cur if old is None else {r: min(cur.get(r, FAR), old.get(r, FAR)) for r in cur.keys() | old.keys()}
            if new != old:
                state[j] = new
                work.append(j)
    return state


def check_distances(code):
    """Violations [(address, instruction, registers)] of the distances around the matrix instructions of one kernel."""
    succ, n = successors(code), len(code)
    info = []
    for _, op, args in code:
        part = args.split(",")
        # a register pair or quad is one operand: [lo:hi] has no comma
        info.append((op.startswith("v_mfma"), op.startswith("v_") and not op.startswith(("v_mfma", "v_cmp")),
                     regs(part[0]), [regs(x) for x in part[1:]],
                     4 if op.startswith("v_mfma") else int(part[0], 0) + 1 if op == "s_nop" else 1))

    def walk(mine, need):
        def step(i, cur):
            cost = info[i][4]
            cur = {r: k + cost for r, k in cur.items() if k + cost < need}
            for r in info[i][2]:
                cur.pop(r, None)
            if info[i][mine]:
                cur.update((r, 0) for r in info[i][2])
            return cur
        return _flow(n, succ, {}, step)
    bad = []
    for i, (before, after) in enumerate(zip(walk(1, 2), walk(0, 11))):
        mfma, _, dst, src, _ = info[i]
        hit = set()
        if mfma and before is not None:
            hit |= set().union(*src) & before.keys()
        if after:
            named = dst.union(*src)
            if mfma and len(src) == 3 and src[2] == dst:
                named = src[0] | src[1]
            hit |= named & after.keys()
        if hit:
            bad.append((code[i][0], " ".join(code[i][1:]), sorted(hit)))
    return bad


def check_library(lib, pattern="."):
    """{kernel: (violations, LDS reads)} of every kernel whose name matches."""
    out = {}
    with tempfile.TemporaryDirectory() as tmp:
        for co in code_objects(lib, tmp):
            listing = subprocess.run([f"{LLVM}/llvm-objdump", "-d", co], capture_output=True, text=True, check=True).stdout
            for name, code in functions(listing).items():
                if code and re.search(pattern, name):
                    bad, reads = check(code)
                    out[name] = (bad + (check_distances(code) if ASM_MFMA.search(name) else []), reads)
    return out


if __name__ == "__main__":
    args = sys.argv[1:]
    lib = args[0] if args else os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "diffusionmodel_amd",
                                            "libldm_hip.so")
    found = check_library(lib, args[1] if len(args) > 1 else ".")
    for name, (bad, reads) in sorted(found.items()):
        print(f"{name[:100]:100s} {reads:5d} LDS reads, {len(bad)} violations")
        for addr, ins, r in bad[:10]:
            print(f"    {addr:x}: {ins}   {r}")
    sys.exit(1 if any(bad for bad, _ in found.values()) else 0)
