"""Generated operator kernels on the CPU: the text that hipRTC would compile, built for the host over
wave_host.hpp, which stands in for the cross-lane operations, the matrix products, LDS and the barriers.
Reads and writes outside a buffer, an LDS array or an int's range end the run with a message."""
import hashlib
import os
import re
import subprocess
import threading

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
COMPILER = "/opt/rocm/llvm/bin/clang++"
FLAGS = ["-O1", "-std=c++17", "-mf16c", "-w", "-ffp-contract=off",
         # an index past its array and an int past its range end the run with SIGILL
         "-fsanitize=array-bounds,signed-integer-overflow,shift-exponent", "-fsanitize-trap=all"]


def available():
    return os.path.exists(COMPILER)


def constants(source):
    return {m[1]: int(m[2]) for m in re.finditer(r"constexpr (?:int|long long) (\w+) = (-?\d+)(?:LL)?;", source)}


def _swap(text, old, new, times=None):
    n = text.count(old)
    assert n and times in (None, n), f"{n} times in the kernel's text: {old}"
    return text.replace(old, new)


def host_text(source):
    """The kernel behind the shared prelude, with what only the GPU has put in host terms."""
    at = min(i for i in (source.find("// storage codes"), source.find("\nconstexpr ")) if i >= 0)
    text = source[at:]
    text = text.replace("__attribute__((address_space(1)))", "").replace("__attribute__((address_space(3)))", "")
    ring = ""
    if "lds.ring" in text:
        # a lane's LDS address is 32 bits there
        text = _swap(text, "__shared__ struct {\n  __attribute__((aligned(1024)))", "static struct Lds {\n  __attribute__((aligned(1024)))", 1)
        text = _swap(text, "} lds;", "}& lds = *(Lds*)(((size_t)mmap(0, sizeof(Lds) + 8192, PROT_READ | PROT_WRITE,"
                                     " MAP_PRIVATE | MAP_ANONYMOUS | MAP_32BIT, -1, 0) + 1023) / 1024 * 1024);", 1)
        text = re.sub(r'asm volatile\("s_waitcnt vmcnt\(%0\)\\n\\ts_barrier" ::"n"\((.*?)\) : "memory"\)', r"wh::turn_barrier(\1)", text)
        text = _swap(text, 'asm volatile("s_waitcnt vmcnt(0)\\n\\ts_barrier" ::: "memory")', "wh::turn_barrier(0)", 1)
        text = re.sub(r'asm volatile\("" : "\+v"\([^;]*\)\);', ";", text)

        def reads(m):
            operands = re.findall(r'"=&v"\((.*?)\)', m[0])
            offsets = re.findall(r'"n"\((\w+)\)', m[0])
            body, n = re.findall(r"ds_read_b64_tr_b16 %(\d+), %(\d+) offset:%(\d+)", m[0]), len(operands)
            assert len(body) == n and m[0].rstrip().endswith('"memory");') and "lgkmcnt(0)" in m[0]
            return "".join("wh::transposed((%s) + %s, %s);" % ("even" if int(a) == n else "even ^ 32u", offsets[int(o) - n - 2], operands[int(r)])
                           for r, a, o in body)
        text = re.sub(r'asm volatile\("ds_read_b64_tr_b16.*?;', reads, text, flags=re.S)
        ring = "ring_lo = (const char*)lds.ring, ring_hi = ring_lo + sizeof lds.ring;"
    assert "asm volatile" not in text, text[text.find("asm volatile"):][:200]
    name = re.search(r'extern "C" __global__ void __launch_bounds__\([^)]*\) (\w+)\(Args a\)', text)[1]
    return (f'#include "{HERE}/wave_host.hpp"\n{text}\n#define KERNEL {name}\n#define RING {ring}\n#include "{HERE}/wave_host_main.hpp"\n')


def build(source, folder, math=True, change=lambda text: text):
    """The executable of a kernel's text, made once per text in `folder`."""
    text = change(host_text(source))
    headers = "".join(open(os.path.join(HERE, n)).read() for n in ("wave_host.hpp", "wave_host_main.hpp"))
    exe = os.path.join(folder, "k" + hashlib.sha256((text + headers + str(math)).encode()).hexdigest()[:20])
    if not os.path.exists(exe):
        mine = exe + f".{threading.get_ident()}"
        with open(mine + ".cpp", "w") as f:
            f.write(text)
        p = subprocess.run([COMPILER, *FLAGS, *([] if math else ["-DWH_NO_MATH"]), mine + ".cpp", "-o", mine], capture_output=True, text=True)
        assert p.returncode == 0, p.stderr[:4000]
        os.replace(mine, exe)
    return exe


def run(exe, folder, grid, operands, order=0, limit=300):
    """operands: bytes (read) or bytearrays (written back) in the order of the kernel's Args. Returns
    what stopped the run, or None."""
    words = [exe, str(grid), str(order)]
    for i, o in enumerate(operands):
        path = os.path.join(folder, f"operand{i}")
        with open(path, "wb") as f:
            f.write(o)
        words += [path, str(len(o)), "w" if isinstance(o, bytearray) else "r"]
    p = subprocess.run(words, capture_output=True, text=True, timeout=limit)
    if p.returncode:
        return p.stderr.strip() or f"exit status {p.returncode}"
    for i, o in enumerate(operands):
        if isinstance(o, bytearray):
            with open(os.path.join(folder, f"operand{i}"), "rb") as f:
                o[:] = f.read()
    return None


def attention_operands(c, q, kc, vc, tables, starts, past, out_bytes):
    """Operands of the matrix-core attention with constants `c`: its inputs as bytes, then output, scratch
    (NaN) and counters (0). The grid too."""
    u32 = lambda x: np.ascontiguousarray(np.asarray(x, np.int64) & 0xFFFFFFFF, dtype=np.uint32).tobytes()  # noqa: E731
    o, counts = bytearray(b"\xa5" * out_bytes), bytearray(c["COUNTS"] * c["NKV"] * 4) if "COUNTS" in c else None
    first = [q, kc, vc, u32(tables), u32(starts), u32(past), o]
    if counts is None:
        return first, (c["T"] * c["NH"] + 3) // 4
    rows = c["T"] * c["REP"]
    tiles = rows // c["PR"] + min(c["B"], c["T"], rows // (c["DR"] + 1)) if rows > c["DR"] else 0
    part = bytearray(b"\xff" * (c["NKV"] * c["SLOTS"] * (c["HD"] + 2) * 4))
    return first + [part, counts], c["NKV"] * (c["FEW_GROUPS"] + max(tiles, c["PSPLIT"]))
