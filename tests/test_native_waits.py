"""How the native sources wait, read from them: what a wrong order or a divided warp does shows on a device only as a rare hang."""
import re

import pytest

from batchspec_b200.csrc.build import CSRC

WHOLE_WARP = "__all_sync(0xffffffffu, "


@pytest.mark.parametrize("name", ["gemm_fp8.cu", "moe_layer.cu"])
def test_a_warp_learns_one_answer_from_a_wait(name):
    """A wait that runs out is answered with a refusal.  In these kernels a whole warp waits, and what follows is for whole warps (reads of tensor
    memory, ``__syncwarp``), so all lanes have to go on or all to leave: ``warp_wait``, ``warp_wait_short``, or a vote around the wait."""
    text = (CSRC / name).read_text()
    waits = list(re.finditer(r"\bmbar_wait(?:_short)?(?:<\w+>)?\(", text))
    alone = [text.count("\n", 0, m.start()) + 1 for m in waits if not text[:m.start()].endswith(WHOLE_WARP)]
    assert alone == []
    assert len(re.findall(r"\bwarp_wait(?:_short)?\(", text)) > 5
    helpers = (CSRC / "tma.cuh").read_text()
    for short in ("", "_short"):
        body = re.search(r"bool warp_wait" + short + r"\([^{]*\{([^}]*)\}", helpers).group(1)
        assert body.strip().startswith("return " + WHOLE_WARP + "mbar_wait" + short + "(")


def kernels_with_tensor_memory():
    """(file, kernel, its text) of every kernel that takes tensor memory."""
    found = []
    for path in sorted(CSRC.glob("*.cu")):
        for part in path.read_text().split("__global__")[1:]:
            if "tcgen05.alloc" in part:
                found.append(pytest.param(part, id=path.name + ":" + re.search(r"(\w+_kernel)\(", part).group(1)))
    return found


@pytest.mark.parametrize("text", kernels_with_tensor_memory())
def test_tensor_memory_is_held_before_the_next_kernel_may_start(text):
    """``tcgen05.alloc`` waits without a limit.  A kernel that lets its successor start before all of its own CTAs hold their columns could wait
    for columns that a CTA of the successor holds, which waits for this kernel's end."""
    starts = [m.start() for m in re.finditer(r"pdl_(?:launch_dependents|prologue|prologue_late)\(", text)]
    assert not starts or min(starts) > text.index("tcgen05.alloc")
