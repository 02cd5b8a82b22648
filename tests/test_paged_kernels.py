"""What the paged cache's kernels rely on that no run shows reliably: read from the assembly that the library's own
flags give (gfx950; needs hipcc, no GPU)."""

import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from poly_attention import _build

SOURCES = ["pa_paged_tiles_bf16", "pa_paged_tiles_f16", "pa_paged_bf16", "pa_paged_f16", "pa_paged_f32", "pa_paged", "pa_page"]
COPY = re.compile(r"v_accvgpr_(write|read)_b32|v_mov_b(32|64)_e\d+ v\S+ v")
VECTOR = ("v_", "ds_", "global_", "buffer_", "scratch_", "flat_")
TO_SCALAR = ("v_readlane", "v_readfirstlane", "v_writelane", "v_cmp")


def functions(lines):
    """{name: its lines without comments, but for the marks of inline assembly}."""
    out, body = {}, None
    for line in lines:
        if re.match(r"_Z\w+:", line):
            body = out[line.split(":")[0]] = []
        elif body is not None:
            if ".end_amdhsa_kernel" in line:
                body = None
                continue
            mark = re.search(r"#ASM(START|END)", line)
            text = mark[0] if mark else line.split(";")[0].strip()
            if text and (not text.startswith(".") or text.endswith(":")):
                body.append(text)
    return out


def copies_without_lanes(body):
    """Register copies at the target of a branch that is taken when no lane is active, ahead of the instruction that switches
    lanes on again: they copy nothing on that path."""
    at = {text[:-1]: i for i, text in enumerate(body) if text.endswith(":")}
    bad = []
    for target in {text.split()[1] for text in body if text.startswith("s_cbranch_execz")} & set(at):
        vectors = []
        for text in body[at[target] + 1:]:
            op = text.split()[0]
            if op.startswith("s_") and "exec" in text:
                if text.startswith("s_or_b64 exec, exec") and all(COPY.match(v) for v in vectors):
                    bad += vectors
                break
            if op in ("s_endpgm", "s_branch", "s_setpc_b64") or op.startswith("s_cbranch"):
                break
            if op.startswith(VECTOR) and not op.startswith(TO_SCALAR):
                vectors.append(text)
    return bad


def registers(text):
    out = {int(m) for m in re.findall(r"\bs(\d+)\b", text)}
    for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        out |= set(range(int(a), int(b) + 1))
    return out


def short_waits(body):
    """Loads in inline assembly that read a scalar register fewer than five wait states after a vector instruction wrote it."""
    bad, last, inline = [], [], False  # last: (what a vector instruction wrote, wait states)
    for text in body:
        if text.startswith("#ASM"):
            inline = text == "#ASMSTART"
            continue
        if text.endswith(":"):
            continue
        op, _, args = text.partition(" ")
        if inline and op.startswith("buffer_load"):
            need, states = registers(args), 0
            for wrote, wait in reversed(last):
                if states >= 5:
                    break
                if wrote & need:
                    bad.append(text)
                    break
                states += wait
        last = last[-11:] + [(registers(args.split(",")[0]) if op.startswith("v_") else set(),
                              int(args, 0) + 1 if op == "s_nop" else 1)]
    return bad


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    try:
        hipcc = _build.hipcc()
    except RuntimeError:
        pytest.skip("no hipcc")
    out = tmp_path_factory.mktemp("paged")

    def compiled(name):
        path = out / f"{name}.s"
        subprocess.run([hipcc, *_build.COMMON_FLAGS, "--cuda-device-only", "-S", str(_build.SRC_DIR / f"{name}.hip"), "-o", str(path)],
                       check=True, capture_output=True, text=True)
        return functions(path.read_text().splitlines())

    with ThreadPoolExecutor(len(SOURCES)) as pool:
        return dict(zip(SOURCES, pool.map(compiled, SOURCES)))


@pytest.mark.parametrize("source", SOURCES)
def test_no_copies_without_lanes(kernels, source):
    """The first k_paged_tiles faulted the GPU by such copies: addresses were formed from registers that nothing was copied
    to, where a unit had one tile of positions."""
    assert kernels[source]
    bad = {name: found for name, body in kernels[source].items() if (found := copies_without_lanes(body))}
    assert not bad


@pytest.mark.parametrize("source", SOURCES)
def test_direct_loads_wait_for_their_registers(kernels, source):
    """The compiler does not see into the assembly of the direct loads, so it leaves no wait states before it."""
    loads = sum(text.startswith("buffer_load") and " lds" in text for body in kernels[source].values() for text in body)
    assert (loads > 0) == ("tiles" in source)
    bad = {name: found for name, body in kernels[source].items() if (found := short_waits(body))}
    assert not bad


def test_the_checks_find_what_they_look_for():
    copies = """_Zk:
    s_cbranch_execz .LBB0_2
    v_mov_b32_e32 v1, v2
.LBB0_2:
    v_accvgpr_write_b32 a3, v5 ; a copy
    s_or_b64 exec, exec, s[4:5]
    s_endpgm""".splitlines()
    assert copies_without_lanes(functions(copies)["_Zk"]) == ["v_accvgpr_write_b32 a3, v5"]
    assert not copies_without_lanes(functions(copies[:4] + copies[5:])["_Zk"])
    load = ["_Zk:", "    v_readfirstlane_b32 s6, v0", "    s_nop 3", "    ;;#ASMSTART", "    s_mov_b32 m0, s2",
            "    s_nop 0", "    buffer_load_dwordx4 v1, s[4:7], 0 offen lds", "    ;;#ASMEND"]
    assert not short_waits(functions(load)["_Zk"])  # 4 + 1 + 1
    assert short_waits(functions(load[:2] + load[3:])["_Zk"])
