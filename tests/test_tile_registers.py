"""What the tile's kernels (nt_tile.hpp) take for granted of the code made from them, looked up in the built library: an
LDS read issued in one place and waited for in another has its register to itself until then (no instruction reads,
writes, copies or spills it), and the sums of a tile stay in registers. On the CPU, from the library's own disassembly."""
import os
import re
import struct
import subprocess

import pytest

import noetic_rl as nr

TOOLS = "/opt/rocm/llvm/bin"
KERNELS = ("k_readout_stats", "k_readout_g", "k_readout_grad", "k_int8_tiles")

REGISTER = re.compile(r"\b([va])(?:(\d+)\b|\[(\d+):(\d+)\])")
OPCODE = re.compile(r"\s([a-z]\w+)(.*?)//\s*([0-9A-Fa-f]+):[^<]*(?:<\S+?\+0x([0-9a-f]+)>)?")


def registers(text):
    out = set()
    for kind, one, first, last in REGISTER.findall(text):
        out.update(kind + str(i) for i in (range(int(one), int(one) + 1) if one else range(int(first), int(last) + 1)))
    return out


def touched_in_flight(code):
    """[(address, instruction)] that touch a register whose LDS read has not been waited for, and the number of reads;
    `code`: (address, opcode, operands, a branch's target) in order. LDS operations end in their order, so a wait for n
    outstanding leaves the last n; what is outstanding where branches meet is what any of them leaves."""
    starts = {code[0][0]} | {t for _, _, _, t in code if t is not None}
    starts |= {code[k + 1][0] for k in range(len(code) - 1) if code[k][1].startswith(("s_branch", "s_cbranch", "s_endpgm"))}
    blocks, at = {}, None
    for k, (addr, op, args, target) in enumerate(code):
        if addr in starts:
            at = addr
            blocks[at] = ([], [])
        blocks[at][0].append((addr, op, args))
        following = code[k + 1][0] if k + 1 < len(code) else None
        if op.startswith(("s_branch", "s_cbranch")):
            blocks[at][1].append(target)
        if following in starts and not op.startswith(("s_branch", "s_endpgm")):
            blocks[at][1].append(following)
    bad, reads = set(), set()

    def through(block, queue):
        queue = list(queue)
        for addr, op, args in block:
            if op == "s_waitcnt":
                m = re.search(r"lgkmcnt\((\d+)\)", args)
                if m:
                    queue = queue[max(0, len(queue) - int(m.group(1))):]
                continue
            flying = set().union(*queue) if queue else set()
            if registers(args) & flying:
                bad.add((addr, op + args))
            if op.startswith(("ds_read", "ds_bpermute", "ds_permute", "ds_swizzle")):
                queue.append(frozenset(registers(args.split(",")[0])))
                reads.add(addr)
            elif op.startswith(("ds_", "s_load", "s_buffer_load")):
                queue.append(frozenset())
        return tuple(queue)

    state, work = {code[0][0]: ()}, [code[0][0]]
    while work:
        b = work.pop()
        out = through(blocks[b][0], state[b])[-64:]
        for s in blocks[b][1]:
            old = state.get(s)
            n = max(len(out), len(old or ()))
            pad = lambda q: (frozenset(),) * (n - len(q)) + tuple(q)  # noqa: E731
            new = pad(out) if old is None else tuple(x | y for x, y in zip(pad(out), pad(old)))
            if old is None or new != pad(old):
                state[s] = new
                work.append(s)
    return sorted(bad), len(reads)


def listing(text):
    """{function: code} of a disassembly."""
    out, code, base = {}, None, 0
    for line in text.splitlines():
        m = re.match(r"^([0-9a-f]+) <(\S+)>:", line)
        if m:
            base, code = int(m.group(1), 16), []
            out[m.group(2)] = code
            continue
        m = OPCODE.match(line)
        if m and code is not None:
            op = m.group(1)
            branch = op.startswith(("s_branch", "s_cbranch"))
            code.append((int(m.group(3), 16), op, m.group(2), base + int(m.group(4) or "0", 16) if branch else None))
    return out


PLANTED = """
0000000000001000 <k>:
	ds_read_b128 v[0:3], v8    // 000000001000: 00000000
	v_add_f32 v9, v10, v11     // 000000001008: 00000000
	{a}                        // 00000000100C: 00000000
	s_waitcnt lgkmcnt(0)       // 000000001010: 00000000
	v_add_f32 v9, v0, v11      // 000000001014: 00000000
	{b}                        // 000000001018: 00000000
	s_cbranch_scc1 65530       // 00000000101C: 00000000 <k+0x8>
	s_endpgm                   // 000000001020: 00000000
"""


@pytest.mark.parametrize("a,b,bad", [
    ("s_nop 0", "s_nop 0", []), ("v_mov_b32 v20, v2", "s_nop 0", [0x100c]), ("v_mov_b32 v3, v20", "s_nop 0", [0x100c]),
    ("scratch_store_dword off, v0, off", "s_nop 0", [0x100c]), ("ds_read_b32 v1, v8", "s_nop 0", [0x100c]),
    ("s_nop 0", "ds_read_b32 v10, v8", [0x1008]),   # in flight where the loop closes
    ("ds_read_b32 v30, v8", "s_nop 0", [])])
def test_the_check_finds_what_it_is_for(a, b, bad):
    found, _ = touched_in_flight(listing(PLANTED.format(a=a, b=b))["k"])
    assert [addr for addr, _ in found] == bad


@pytest.fixture(scope="module")
def objects(tmp_path_factory):
    if not os.path.exists(f"{TOOLS}/llvm-objdump"):
        pytest.skip("no llvm-objdump")
    data, mark = open(nr.LIB_PATH, "rb").read(), b"__CLANG_OFFLOAD_BUNDLE__"
    folder, out, at = tmp_path_factory.mktemp("objects"), [], data.find(mark)
    while at >= 0:
        n, = struct.unpack_from("<Q", data, at + 24)
        o = at + 32
        for _ in range(n):
            off, size, length = struct.unpack_from("<QQQ", data, o)
            target = data[o + 24:o + 24 + length]
            o += 24 + length
            code = data[at + off:at + off + size]
            if b"gfx950" in target and any(k.encode() in code for k in KERNELS):
                out.append(folder / f"{len(out)}.co")
                out[-1].write_bytes(code)
        at = data.find(mark, at + 24)
    assert len(out) == 2  # the readout's and the 8-bit product's
    return out


def tile_kernels(names):
    return [n for n in names if any(re.search(rf"\d{k}I", n) for k in KERNELS)]


def test_registers_of_reads_in_flight_are_left_alone(objects):
    seen = 0
    for path in objects:
        text = subprocess.run([f"{TOOLS}/llvm-objdump", "-d", str(path)], check=True, capture_output=True, text=True).stdout
        code = listing(text)
        for name in tile_kernels(code):
            bad, reads = touched_in_flight(code[name])
            assert not bad, (name, bad[:5])
            assert reads >= 20, (name, reads)  # (its fragments' at the least)
            seen += 1
    assert seen >= 60


def test_sums_stay_in_registers(objects):
    """A tile's sums are 256 bytes a lane at the least, 1024 of 256 x 256: what a kernel keeps in memory is less."""
    seen = 0
    for path in objects:
        notes = subprocess.run([f"{TOOLS}/llvm-readelf", "--notes", str(path)], check=True, capture_output=True, text=True).stdout
        for name, size in re.findall(r"\.name:\s+(\S+)\n(?:.*\n)*?\s+\.private_segment_fixed_size: (\d+)", notes):
            if tile_kernels([name]):
                assert int(size) < 256, (name, size)
                seen += 1
    assert seen >= 60
