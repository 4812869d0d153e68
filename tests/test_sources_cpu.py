"""Rules of the CUDA sources that no run can show reliably, read from the sources."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "roofline_decoding_b200" / "csrc"
SOURCES = sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")])


def asm_statements(text):
    """The text of every asm statement, by its balanced parentheses."""
    for m in re.finditer(r"\basm\b(?:\s+volatile)?\s*\(", text):
        depth, i, quoted = 1, m.end(), False
        while depth:
            c = text[i]
            if c == '"' and text[i - 1] != "\\":
                quoted = not quoted
            elif not quoted:
                depth += (c == "(") - (c == ")")
            i += 1
        yield text[m.start():i]


def test_loads_from_tensor_memory_wait_in_their_own_statement():
    """tcgen05.ld writes its registers later; only a wait in the same statement keeps the
    compiler from using, moving or spilling them before they are there."""
    seen = 0
    for path in SOURCES:
        for s in asm_statements(path.read_text()):
            if "tcgen05.ld." in s:
                seen += 1
                assert "tcgen05.wait::ld" in s, f"{path.name}: {s[:120]}"
    assert seen > 0


def test_a_prompt_block_that_gives_up_leaves_nothing_in_flight():
    """Before the last barrier and the release of tensor memory: the copy warp waits for each
    buffer's last copy, the MMA lane for its products; and a warp gives up with all its lanes."""
    text = (CSRC / "w4_kv8_prompt.cu").read_text()
    kernel = text[text.index("kv8_prompt_kernel(const AttnP p)"):text.index("int launch_prompt(")]
    end = kernel.index("tc_dealloc")
    copies = kernel.index("bulk_load(")
    drained = kernel.index("wait(&raw_full[i]", copies)
    products = kernel.index("tc_commit(mma_done)")
    assert copies < drained < products < kernel.index("wait_on(mma_done", products) < end
    assert kernel.rindex("__syncthreads", 0, end) > products
    one_lane = kernel[kernel.index("} else if (warp == kMmaWarp && lane == 0) {"):
                      kernel.index("} else if (warp >= kWidenWarp) {")]
    voted = "__all_sync(0xffffffffu, wait_on(bar, parity))"
    assert voted in kernel and kernel.count("wait_on(") == one_lane.count("wait_on(") + 1
    assert not re.search(r"[^_\w]wait\(", one_lane) and "next_item()" not in one_lane
    # which phase of a buffer's barrier its last copy completes
    bufs = 3
    for issued in range(12):
        stage, turn = issued % bufs, (issued // bufs) & 1
        for i in range(bufs):
            of_it = len([k for k in range(issued) if k % bufs == i])  # phases completed or due
            parity = turn if i < stage else turn ^ 1
            assert parity == (of_it - 1) & 1  # of none: the phase before the first, which passes


def test_gemm_warps_give_up_with_all_their_lanes():
    """Loads from tensor memory and the warps' barriers need every lane."""
    text = (CSRC / "w4_gemm.cu").read_text()
    role = text[text.index("- dequant\n    constexpr"):text.index("tc_dealloc")]
    assert role.index("__all_sync") < role.index("break;")
    assert "__any_sync(0xffffffffu, stopped())" in role and role.count("stopped()") == 1


def test_kernels_that_start_before_their_inputs_are_written_make_no_read_only_loads():
    """ld.global.nc and __ldg ask that the memory does not change while the kernel is there; a
    programmatic dependent is there before the kernel in front of it has written it."""
    for path in [CSRC / "w4_gemm.cu", *CSRC.glob("w4_kv8*.cu"), *CSRC.glob("w4_kv8*.cuh")]:
        code = re.sub(r"//[^\n]*", "", path.read_text())
        assert not re.search(r"__ldg|ld\.global\.nc|__restrict__", code), path.name
