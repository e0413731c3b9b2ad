"""Waits that the compiler does not put: the large tiles' MFMAs are inline asm, so what reads their accumulators has to come
a fixed number of instructions later. Read from the built library's gfx950 code, which no output shows reliably."""
import os
import re
import struct
import subprocess

import pytest

OBJDUMP = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")
WAIT = 20   # wait states, more than any MFMA needs before its results are read


def _code_objects():
    import _native
    if not os.path.exists(_native.LIB_PATH) or not os.path.exists(OBJDUMP):
        pytest.skip("library not built, or no llvm-objdump")
    data = open(_native.LIB_PATH, "rb").read()
    at = data.find(b"__CLANG_OFFLOAD_BUNDLE__")
    while at >= 0:
        entry = at + 32
        for _ in range(struct.unpack_from("<Q", data, at + 24)[0]):
            off, size, name = struct.unpack_from("<QQQ", data, entry)
            target, entry = data[entry + 24:entry + 24 + name], entry + 24 + name
            if target.endswith(b"gfx950"):
                yield data[at + off:at + off + size]
        at = data.find(b"__CLANG_OFFLOAD_BUNDLE__", at + 1)


@pytest.fixture(scope="module")
def big(tmp_path_factory):
    """{kernel: [(address, text)]} of every gm_big_kernel."""
    out = {}
    path = str(tmp_path_factory.mktemp("waits") / "code.o")
    for elf in _code_objects():
        if b"gm_big_kernel" not in elf:
            continue
        with open(path, "wb") as f:
            f.write(elf)
        cur = None
        text = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", path], capture_output=True, text=True, check=True).stdout
        for line in text.split("\n"):
            m = re.match(r"^[0-9a-f]+ <(\S+)>:", line)
            if m:
                cur = out.setdefault(m.group(1), []) if "gm_big_kernel" in m.group(1) else None
            elif cur is not None and "//" in line:
                ins, tail = line.split("//", 1)
                cur.append((int(tail.split(":")[0], 16), ins.strip(), tail))
    return out


def _regs(op, kind):
    m = re.match(kind + r"\[(\d+):(\d+)\]$", op) or re.match(kind + r"(\d+)()$", op)
    return set(range(int(m.group(1)), int(m.group(2) or m.group(1)) + 1)) if m else set()


def test_accumulators_are_read_after_the_wait(big):
    assert len(big) == 11   # bf16 and fp16: gate|up, NT, dh, dx, TN; int8
    for name, code in big.items():
        at = {a: k for k, (a, _, _) in enumerate(code)}
        start = code[0][0]
        mfmas = [k for k, (_, i, _) in enumerate(code) if i.startswith("v_mfma")]
        assert len(mfmas) == 256, (name, len(mfmas))
        seen = set()
        for k in mfmas:
            regs = _regs(code[k][1].split()[1].rstrip(","), "a")
            work = [(k + 1, 0)]
            while work:
                j, waited = work.pop()
                if waited >= WAIT or (k, j, waited) in seen:
                    continue
                seen.add((k, j, waited))
                ins = code[j][1]
                op, args = (ins.split(None, 1) + [""])[:2]
                if not op.startswith("v_mfma"):
                    hit = set().union(*(_regs(a.strip(), "a") for a in args.split(","))) & regs
                    assert not hit, (name, code[k][1], ins, waited)
                if op == "s_endpgm":
                    continue
                waited += 1 + (int(args, 0) if op == "s_nop" else 0)
                if op.startswith(("s_cbranch", "s_branch")):
                    to = at[start + int(re.search(r"\+0x([0-9a-f]+)>", code[j][2]).group(1), 16)]
                    work.append((to, waited))
                if op != "s_branch":
                    work.append((j + 1, waited))


def test_asm_names_m0_where_it_writes_it():
    """An asm that sets M0 (the LDS address of direct loads) says so, or the compiler may keep a value of its own there."""
    src = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "glm-flash-lite_amd", "csrc")
    found = 0
    for name in sorted(os.listdir(src)):
        if name.endswith((".hip", ".hpp")):
            with open(os.path.join(src, name)) as f:
                for stmt in re.findall(r"asm volatile\((.*?)\);", f.read(), re.S):
                    if re.search(r"\bm0, %", stmt):
                        found += 1
                        assert '"m0"' in stmt.rsplit(":", 1)[1], (name, stmt)
    assert found


def test_large_tiles_k_loop_has_no_scratch(big):
    """The K loop, two steps of 64 MFMAs, touches no scratch memory; what the kernel spills it spills around its ends."""
    for name, code in big.items():
        at = {a: k for k, (a, _, _) in enumerate(code)}
        start = code[0][0]
        loops = []
        for k, (_, ins, tail) in enumerate(code):
            if ins.startswith(("s_cbranch", "s_branch")):
                to = at[start + int(re.search(r"\+0x([0-9a-f]+)>", tail).group(1), 16)]
                body = [i for _, i, _ in code[to:k + 1]]
                if to < k and sum(i.startswith("v_mfma") for i in body) == 128:
                    loops.append(body)
        body = min(loops, key=len)
        assert not [i for i in body if i.startswith("scratch_")], name
