"""The sums of a team of threads are read sixteen bytes at a time: their place in shared memory carries that alignment in its type,
whatever else a kernel keeps there."""
import subprocess

from ascend_mlir_b200 import build as lib_build

SOURCE = r"""
#include <type_traits>
#include "kernels/block_norm_device.cuh"
using namespace afir::kernels;
static_assert(alignof(TeamScratch) >= 16 && sizeof(TeamScratch) == kTeamScratchFloats * sizeof(float), "16-byte loads");
static_assert(!std::is_invocable<decltype(makeTeam), int, float *>::value, "no buffer of another alignment");
static_assert(kTeamSlice % 4 == 0, "each value's part begins on 16 bytes");
__global__ void kernel(int lanes, float *out) {
  __shared__ char other[5];
  __shared__ TeamScratch scratch;
  Team team = makeTeam(lanes, scratch);
  other[threadIdx.x % 5] = static_cast<char>(team.index);
  float v[1] = {static_cast<float>(threadIdx.x)};
  teamSum(team, v);
  if (team.lane == 0) out[team.index] = v[0] + other[0];
}
"""


def test_alignment_is_part_of_the_type(tmp_path):
    (tmp_path / "team.cu").write_text(SOURCE)
    res = subprocess.run([lib_build.NVCC, *lib_build.NVCC_FLAGS, "-c", str(tmp_path / "team.cu"), "-o", str(tmp_path / "team.o")], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
