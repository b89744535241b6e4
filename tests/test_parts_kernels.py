"""The kernels of listed groups and drafted nodes as the compiler made them (gfx950, no GPU): no register spills, no packed fp32
arithmetic, wait states around inline asm, and no vector memory instruction but the stream's own between the hand-counted waits of the
streaming kernels."""
import re

import pytest

from test_kernel_resources import asm_mfma_hazards, compile_device, kernel_bodies, resources


@pytest.mark.slow
@pytest.mark.parametrize("src,names,least", [("sjk_attend3.hip", ("ext_scalar_kernel", "ext_trellis_kernel", "ext_stream_kernel", "ext_combine"), 28),
                                             ("sjk_select.hip", ("score_kernel", "pick_kernel"), 6), ("sjk_pages.hip", ("accept",), 2)])
def test_no_scratch_no_packed_fp32_no_hazards(src, names, least):
    res = resources(src)
    kernels = [k for k in res if any(n in k for n in names)]
    assert len(kernels) >= least, sorted(res)
    for k in kernels:
        assert res[k].get("ScratchSize [bytes/lane]", -1) == 0, (k, res[k])
    bodies = kernel_bodies(compile_device(src)[1])
    for k in kernels:
        assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", "\n".join(bodies[k])), k
        assert not asm_mfma_hazards(bodies[k]), k


@pytest.mark.slow
def test_streams_have_no_other_vector_memory_instructions():
    bodies = {k: v for k, v in kernel_bodies(compile_device("sjk_attend3.hip")[1]).items() if "ext_stream_kernel" in k}
    assert len(bodies) == 8, sorted(bodies)
    for k, lines in bodies.items():
        waits = [i for i in range(len(lines) - 1) if "ASMSTART" in lines[i] and "s_waitcnt vmcnt(" in lines[i + 1]]
        assert len(waits) >= 8, (k, len(waits))
        foreign = [t.strip() for t in lines[waits[0]:waits[-1]]
                   if t.strip().startswith(("flat_", "scratch_", "buffer_")) or
                   (t.strip().startswith("global_") and "_lds_" not in t.strip().split()[0])]
        assert not foreign, (k, foreign[:4])
