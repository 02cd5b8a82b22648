"""What the drafted step's kernels rely on that no run shows reliably: read from the assembly that the library's
own flags give (gfx950; needs hipcc, no GPU)."""

import re
import subprocess

import pytest

from poly_attention import _build


def assembly(source, kernel, out):
    """The lines of one kernel of csrc/`source`."""
    try:
        hipcc = _build.hipcc()
    except RuntimeError:
        pytest.skip("no hipcc")
    subprocess.run([hipcc, *_build.COMMON_FLAGS, "--cuda-device-only", "-S", str(_build.SRC_DIR / source), "-o", str(out)],
                   check=True, capture_output=True, text=True)
    lines = out.read_text().splitlines()
    start = next(i for i, line in enumerate(lines) if re.match(rf"_ZN2pa\d+{kernel}[^:]*:", line))
    end = next(i for i in range(start, len(lines)) if "s_endpgm" in lines[i])
    return [line.strip() for line in lines[start:end]]


def test_commit_has_read_the_count_at_its_barrier(tmp_path):
    """The workgroup that draws a row's last ticket writes counts[b]; the others draw theirs behind the barrier.
    So no load of a wave may be on its way at the barrier: a barrier does not wait for them by itself."""
    body = assembly("pa_draft.hip", "k_draft_commit", tmp_path / "draft.s")
    ticket = next(i for i, line in enumerate(body) if line.startswith("global_atomic_add"))
    barrier = next(i for i, line in enumerate(body) if line.startswith("s_barrier"))
    assert barrier < ticket
    loads = [i for i, line in enumerate(body[:barrier]) if line.startswith(("global_load", "flat_load", "buffer_load"))]
    waits = [i for i, line in enumerate(body[:barrier]) if line.startswith("s_waitcnt") and "vmcnt(0)" in line]
    assert loads and waits and max(waits) > max(loads)
