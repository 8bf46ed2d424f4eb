"""CPU: rules that the 4-bit kernels' early starts rest on, read from their sources."""
import re
from pathlib import Path

import pytest

KERNELS = Path(__file__).resolve().parent.parent / "csrc" / "kernels"


def kernel_bodies(name):
    """(kernel name, body without comments) of every __global__ function of a source file."""
    text = re.sub(r"//[^\n]*", "", (KERNELS / name).read_text())
    for m in re.finditer(r"__global__ void(?: __launch_bounds__\([^{;]*?\))?\s+(\w+)\([^{;]*?\) \{", text):
        depth, i = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            i += 1
        yield m.group(1), text[m.end():i]


@pytest.mark.parametrize("name,kernels", [("fp4_gemm.cu", {"fp4_gemm_kernel", "fp4_gemm_pair_kernel"}),
                                          ("fp4_moe.cu", {"fp4_moe_up_kernel", "fp4_moe_down_kernel"})])
def test_tensor_memory_is_taken_behind_an_unconditional_wait(name, kernels):
    """A kernel that is scheduled beside the one before it and holds tensor memory while it waits for that one's end would keep
    it from its own allocation for good.  What lies before a launch in its stream is not known, not even behind a launch of the
    same call: another host thread may share the stream."""
    seen = set()
    for kernel, body in kernel_bodies(name):
        for alloc in re.finditer(r"tmem_alloc\(|tcgen05\.alloc", body):
            seen.add(kernel)
            waits = [line for line in body[:alloc.start()].splitlines() if line.strip() == "pdl_wait();"]
            assert waits, f"{kernel} takes tensor memory before an unconditional pdl_wait()"
            assert "pdl_launch();" not in body[:alloc.start()], f"{kernel} lets its dependents start before it has its tensor memory"
    assert seen == kernels


def test_the_expander_lets_nothing_start_early():
    """Its output may be the weights of the next kernel, and the decode GEMVs fetch weights before they wait."""
    bodies = dict(kernel_bodies("fp4.cu"))
    assert "pdl_launch" in bodies["fp4_quantize_kernel"] and "pdl_wait();" in bodies["fp4_dequantize_kernel"]
    assert "pdl_launch" not in bodies["fp4_dequantize_kernel"]


def test_reading_the_status_words_erases_no_report_that_it_has_not_seen():
    text = re.sub(r"//[^\n]*", "", (KERNELS / "fp4.cu").read_text())
    body = text[text.index("FB_API int fb_fp4_status"):]
    body = body[:body.index("\n}")]
    clear = body.index("cudaMemsetAsync")
    assert body.index("cudaStreamSynchronize") < clear and "host[0]" in body[:clear]
