"""64-bit shifts of the built library's gfx950 code: none takes its amount from the last vector register of its wave's
allocation (eight registers at a time). The matrix products of the 16-bit experts gave wrong values now and then while they
had such a shift, and no other difference; the compiler does place amounts there."""
import re
import subprocess

LLVM = "/opt/rocm/llvm/bin/"
SHIFT = re.compile(r"\s(v_(?:lshlrev_b64|lshrrev_b64|ashrrev_i64)\S*)\s+v\[\d+:\d+\], v(\d+),")


def last_registers(notes):
    """kernel name -> the number of its allocation's last register, of a code object's notes."""
    out = {}
    for block in notes.split("- .agpr_count:")[1:]:
        name, count = re.search(r"\.name:\s+(\S+)", block), re.search(r"\.vgpr_count:\s+(\d+)", block)
        if name and count:
            out[name[1]] = (int(count[1]) + 7) // 8 * 8 - 1
    return out


def bad_shifts(listing, last):
    name, found = None, []
    for line in listing.splitlines():
        m = re.match(r"[0-9a-f]{16} <(.*)>:$", line)
        if m:
            name = m[1]
        m = SHIFT.search(line)
        if m and name in last and int(m[2]) == last[name]:
            found.append(f"{name}: {line.strip()}")
    return found


def test_the_check_sees_a_shift():
    notes = "- .agpr_count: 0\n .name: k\n .vgpr_count: 126\n"
    assert last_registers(notes) == {"k": 127}
    for register, bad in ((127, 1), (126, 0)):
        listing = f"0000000000001000 <k>:\n\tv_lshlrev_b64 v[2:3], v{register}, v[4:5]  // 0000: 00\n"
        assert len(bad_shifts(listing, last_registers(notes))) == bad


def test_no_shift_by_the_last_register(tmp_path):
    import gfr_moe
    lib = tmp_path / "libgfr_moe.so"
    lib.write_bytes(open(gfr_moe.LIB_PATH, "rb").read())
    subprocess.run([LLVM + "llvm-objdump", "--offloading", lib], check=True, capture_output=True, cwd=tmp_path)
    code = sorted(p for p in tmp_path.iterdir() if p.name.endswith("gfx950"))
    assert code
    kernels, bad = 0, []
    for p in code:
        last = last_registers(subprocess.run([LLVM + "llvm-readelf", "--notes", p], check=True, capture_output=True, text=True).stdout)
        kernels += len(last)
        text = subprocess.run([LLVM + "llvm-objdump", "-d", "--no-show-raw-insn", p], check=True, capture_output=True, text=True).stdout
        bad += bad_shifts(text, last)
    assert kernels > 50
    assert not bad, "\n".join(bad)
