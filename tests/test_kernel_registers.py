"""Registers of kernels whose speed hangs on how many workgroups share a compute unit (hipcc cross-compiles here: no GPU needed)."""
import os
import re
import subprocess

from rllama_amd import build

ATTN_ROWS = """
#include "kernels.h"
#include "longctx.h"
#include "attn_rows_device.h"
namespace rlh {
__global__ __launch_bounds__(kAwThreads) void kernel(AttnCutParams p) {
    __shared__ RowsShared<64> shared;
    attn_rows<half_t, half_t, half_t, 64>(WindowView(p), shared, blockIdx.z, blockIdx.y, blockIdx.x);
}
}
"""


def compiled(source, out):
    """[(name, values of the compiler's notes)] of a source file's kernels."""
    flags = [f for f in build.FLAGS if f != "-fPIC"]
    subprocess.run([build.HIPCC, *flags, "--cuda-device-only", "-S", "-I", build.CSRC, str(source), "-o", str(out)], check=True, capture_output=True)
    notes = re.findall(r"- \.agpr_count:(.*?)\.wavefront_size", out.read_text(), re.S)
    assert notes
    return [(re.search(r"\.name:\s+(\S+)", n).group(1), {k: int(v) for k, v in re.findall(r"\.(\w+):\s+(\d+)\n", n)}) for n in notes]


def test_three_workgroups_of_attention_rows_fit_a_compute_unit(tmp_path):
    """f16 rows and planes, heads of 64: eight wavefronts a workgroup, two of them on each SIMD of 512 registers, so 80 at most."""
    src = tmp_path / "rows.hip"
    src.write_text(ATTN_ROWS)
    (_, notes), = compiled(src, tmp_path / "rows.s")
    assert notes["vgpr_count"] <= 80 and notes["private_segment_fixed_size"] == 0


def test_log_probabilities_keep_their_rows_in_registers(tmp_path):
    """No kernel spills to scratch memory, those for rows of any length among them."""
    for name, notes in compiled(os.path.join(build.CSRC, "token_logprobs.hip"), tmp_path / "logprobs.s"):
        assert notes["private_segment_fixed_size"] == 0 and notes["vgpr_spill_count"] == 0, name
