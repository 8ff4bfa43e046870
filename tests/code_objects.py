"""The kernels in a code object that was built here: their instructions and resources."""

import os
import re
import subprocess

LLVM = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin")


def _tool(name, *args):
    return subprocess.run([os.path.join(LLVM, name), *args], capture_output=True, text=True, check=True).stdout


def kernels(path):
    """{name: [(address, instruction, address that it branches to or None)]}"""
    out, code = {}, None
    for line in _tool("llvm-objdump", "-d", "--no-show-raw-insn", path).splitlines():
        head = re.match(r"^([0-9a-f]+) <(.*)>:", line)
        if head:
            code, start = out.setdefault(head.group(2), []), int(head.group(1), 16)
            continue
        m = re.match(r"\s+(\S.*?)\s*//\s*([0-9A-Fa-f]+):(.*)", line)
        if m and code is not None:
            to = re.search(r"<[^>]*\+0x([0-9a-f]+)>", m.group(3))
            code.append((int(m.group(2), 16), m.group(1), start + int(to.group(1), 16) if to else None))
    return out


def scratch_bytes(path):
    """{kernel name: bytes of scratch memory of a lane}, spilled registers among them."""
    name, out = None, {}
    for line in _tool("llvm-readelf", "--notes", path).splitlines():
        m = re.match(r"\s+\.(name|private_segment_fixed_size):\s+(\S+)", line)
        if m and m.group(1) == "name":
            name = m.group(2)
        elif m and name is not None:
            out[name] = int(m.group(2))
    return out


def ahead_of_restore(code):
    """Vector instructions behind the end of a branch of some lanes, ahead of the instruction that lets the
    other lanes go on: what they write is lost for those."""
    at = {a: k for k, (a, _, _) in enumerate(code)}
    found = []
    for k, (_, text, to) in enumerate(code):
        if not text.startswith("s_cbranch_execz") or to not in at:
            continue
        saved = next((m.group(1) for _, t, _ in reversed(code[max(0, k - 40):k])
                      if (m := re.match(r"s_\w+_saveexec_b64 (s\[\d+:\d+\]|vcc)|s_mov_b64 (s\[\d+:\d+\]), exec", t))), None)
        between = []
        for _, t, _ in code[at[to]:at[to] + 60]:
            if t.startswith("s_or_b64 exec, exec, "):
                if saved and t.endswith(saved):
                    found += between
                break
            if re.match(r"s_(c?branch|endpgm|barrier)|s_\w+ exec", t):
                break
            if re.match(r"(v|ds|global|scratch|buffer|flat)_", t) and not re.match(r"v_(readlane|writelane|readfirstlane)", t):
                between.append(t)
    return found
