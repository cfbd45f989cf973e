"""Rules that the attention kernel of k_serve_attn_tc.cu has to keep and that no run shows: read from its source."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "tensorlisp_b200" / "csrc"
TEXT = (CSRC / "k_serve_attn_tc.cu").read_text()


def conditions(text, at):
    """The conditions of the blocks around a place of the source, from the outermost in ("else": of an if without another condition)."""
    stack, begin = [], 0
    for m in re.finditer(r"[{};]", text[:at]):
        if m.group() == "{":
            stack.append(re.sub(r"\s+", " ", re.sub(r"//[^\n]*", "", text[begin:m.start()])).strip())
        elif m.group() == "}":
            stack.pop()
        begin = m.end()
    return stack


def test_register_shares_are_set_by_whole_warpgroups():
    """All threads of a warpgroup have to execute the same setmaxnreg: it stands under conditions that are the same for four warps in a row."""
    places = [m.start() for m in re.finditer(r'asm volatile\("setmaxnreg', TEXT)]
    assert len(places) == 2
    for at in places:
        roles = [c for c in conditions(TEXT, at) if re.match(r"(if|else|for|while)\b", c)]
        assert roles in (["if (warp < 4)"], ["else"]), roles
    assert TEXT.index('"setmaxnreg.dec') < TEXT.index('"setmaxnreg.inc')


def test_every_wait_inside_the_roles_is_bounded():
    """Once a wait has given up, warps leave their roles at different places: between the first role and the barrier in front of the kernel's end nothing
    may wait for a number of threads without a limit, and what is looked at of the others' failure has to be the same for a whole warp."""
    a, b = TEXT.index('"setmaxnreg.dec'), TEXT.index("// only after a wait has given up")
    roles = TEXT[TEXT.index("auto next = [&]"):b]
    assert a < b and "bar.sync" not in roles and "barrier.sync" not in roles and "__syncthreads" not in roles
    looks = re.findall(r"[^\n;{]*\*fail\b[^\n]*", roles)
    assert looks and all("__any_sync(0xffffffffu, *fail" in x for x in looks), looks


def test_a_launch_that_does_not_fit_turns_the_kernel_off():
    """Registers and shared memory (static and dynamic, each instance's own) are looked at where the kernel is set up, and so is whether that worked:
    calls then go to the plain kernel instead of failing at the launch."""
    body = TEXT[TEXT.index("static void sat_configure()"):TEXT.index("void serve_attn_tc_configure()")]
    assert "numRegs" in body and "sharedSizeBytes" in body and "cudaDevAttrMaxSharedMemoryPerBlockOptin" in body
    assert not re.search(r"^\s*cuda\w+\(.*\);$", body.replace("cudaGetLastError();", ""), re.M), "a result that nobody looks at"
    assert "g_sat_fits = false" in body and "!g_sat_fits" in TEXT[TEXT.index("bool serve_attn_tc_supported"):]
