"""What the source of the attention over shared pages has to say for the hardware to keep it: whole warps at tensor memory, fences where it
is handed over, tensor memory before the next kernel may start.  A missing one shows in no run that happens to go well."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cyb_b200", "csrc")


def kernel():
    text = open(os.path.join(CSRC, "attn_shared.cu")).read()
    return text[text.index("attn_tile_kernel(const qeng_shared_attn p"):text.index("// ---- a row's own pages")]


def softmax():
    text = kernel()
    return text[text.index("// ===== softmax"):]


def bare(text):
    return re.sub(r"//[^\n]*", "", text)


def test_warps_are_whole_before_they_read_tensor_memory():
    """tcgen05.ld and .st need a whole warp.  Where a condition of the lane stands in front (one lane arrives at a barrier, some references
    move, some rows attend a key, some have results), only __syncwarp() or a vote says that the lanes are together again."""
    text = bare(softmax())
    assert re.search(r"scores = \[&\]\(int half\) \{\s*__syncwarp\(\);\s*tmem_ld64\(", text) and text.count("tmem_ld64(") == 1
    moved = text[text.index("if (moved) m_run = mx;"):text.index("const float off =")]
    assert moved.count("tmem_ld32(") == 2 and moved.count("__syncwarp();") == 2
    assert re.search(r"if \(j > 0\) \{\s*__syncwarp\(\);", moved) and re.search(r"st_wait\(\);\s*__syncwarp\(\);", moved)
    infinite = text[text.index("const bool on ="):text.index("if (edge && two) mbar_arrive")]
    assert re.search(r"if \(on\) \{[^}]*\}\s*\}\s*__syncwarp\(\);\s*tmem_st32\(", infinite)
    results = text[text.index("const bool result ="):]
    assert results.count("tmem_ld32(") == 1 and re.search(r"__syncwarp\(\);\s*tmem_ld32\(", results)
    assert results.rindex("__syncwarp();") > results.rindex("dst[d * step]")


def test_tensor_memory_changes_hands_between_fences():
    text = bare(softmax())
    waits = [m.end() for m in re.finditer(r"wait_warp\(smem_u32\(sh\.[so]done \+ x\)", text)]
    assert len(waits) == 2
    for at in waits:
        rest = text[at:]
        assert rest.index("fence_after();") < re.search(r"tmem_(ld|st)\d", rest).start()
    for m in re.finditer(r"mbar_arrive\(smem_u32\(&sh\.pready", text):
        before = text[:m.start()]
        assert before.rindex("st_wait();") < before.rindex("fence_before();") < before.rindex("__syncwarp();")
        assert before.rindex("tmem_st16(") < before.rindex("st_wait();")
    mma = bare(kernel()[kernel().index("// ===== MMA issue"):kernel().index("// ===== values that are not finite")])
    for m in re.finditer(r"umma_ts\(", mma):
        before = mma[:m.start()]
        assert before.rindex("mbar_wait(smem_u32(&sh.pready") < before.rindex("fence_after();")


def test_tensor_memory_is_held_before_the_next_kernel_may_start():
    text = bare(kernel())
    assert text.count("griddepcontrol.launch_dependents") == 1 and re.search(r"tmem_alloc\([^}]*griddepcontrol\.launch_dependents", text)
    end = text[text.rindex("fence_before();"):]
    assert end.index("__syncthreads_or(") < end.index("tmem_free(")
