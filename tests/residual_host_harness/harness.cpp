// Drives flagcx_amd/csrc/host_residual.cpp on the CPU, for tests of the split of a block end's gradient
// over teams and of its workspace size.  The launchers that the library would call are replaced by ones
// that note what they are given; the harness then walks every team's rows the way the kernel does.
// Reads lines "rows dim gate gaterows", prints the workspace's bytes for each, and aborts with the reason
// where a row has no team or two, or a partial row lies outside of the workspace.
#include "../../include/flagcx_amd.h"
#include "../../flagcx_amd/csrc/residual.h"

#include <cstdio>
#include <cstdlib>
#include <vector>

namespace flagcx_amd {

static NormBackward seen;
static int calls = 0;

#define NORM(a, r)                                                               \
  int launchNormForward_##a##_##r(const NormForward &, hipStream_t) { return 0; } \
  int launchNormBackward_##a##_##r(const NormBackward &b, hipStream_t) {          \
    seen = b;                                                                    \
    calls++;                                                                     \
    return 0;                                                                    \
  }
NORM(6, 6) NORM(6, 7) NORM(7, 7) NORM(9, 9) NORM(9, 7)
#define EMBED(t, o)                                                             \
  int launchEmbedding_##t##_##o(const EmbedCall &, hipStream_t) { return 0; }    \
  int launchEmbeddingGrad_##t##_##o(const EmbedGradCall &, hipStream_t) { return 0; }
EMBED(6, 6) EMBED(6, 7) EMBED(7, 6) EMBED(7, 7) EMBED(7, 9) EMBED(9, 7) EMBED(9, 9)
uint64_t embedGradWorkspace(uint64_t, uint64_t, uint64_t) { return 0; }
void setLastError(const char *text) { fprintf(stderr, "%s\n", text); }

} // namespace flagcx_amd

extern "C" hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
extern "C" const char *hipGetErrorString(hipError_t) { return ""; }

using namespace flagcx_amd;

static void die(const char *what, size_t rows, size_t dim, size_t gaterows) {
  fprintf(stderr, "%s: rows %zu dim %zu gaterows %zu\n", what, rows, dim, gaterows);
  exit(1);
}

int main() {
  size_t rows, dim, gaterows;
  int gate;
  auto at = [](uint64_t n) { return (void *)(uintptr_t)(n << 40); }; // made-up addresses, far apart
  std::vector<uint8_t> taken;
  while (scanf("%zu %zu %d %zu", &rows, &dim, &gate, &gaterows) == 4) {
    flagcxLocalBlockEnd end = {};
    end.rows = rows;
    end.dim = dim;
    end.norms = FLAGCX_LOCAL_NORM_POST | FLAGCX_LOCAL_NORM_PRE;
    end.datatype = end.residualtype = end.weighttype = flagcxFloat32;
    end.scale = 1.0f;
    end.eps = 1e-6f;
    end.postweight = at(1);
    end.preweight = at(2);
    end.gate = gate ? at(3) : nullptr;
    end.gaterows = gaterows;
    size_t bytes = 0;
    if (flagcxLocalReduceNormBackwardWorkspace(&end, &bytes) != flagcxSuccess) die("no size", rows, dim, gaterows);
    hipStream_t none = nullptr;
    calls = 0;
    const flagcxResult_t r = flagcxLocalReduceNormBackward(
        &end, at(4), 0, at(5), 0, at(6), 0, at(7), 0, at(8), 0, at(9), 0, at(10), at(11), gate ? at(12) : nullptr, 0,
        bytes ? at(13) : nullptr, bytes, (flagcxStream_t)&none);
    if (r != flagcxSuccess || calls != 1) die("no launch", rows, dim, gaterows);
    const NormTeams &t = seen.t;
    if (t.teams != t.parts * t.abreast) die("teams", rows, dim, gaterows);
    const bool partial = seen.dgate && seen.c.gateRows != 1 && t.parts > 1;
    uint64_t partials = 2ull * t.teams; // partial rows that are written: dW1 and dW2 of every team
    taken.assign(rows, 0);
    for (uint64_t me = 0; me < t.teams; me++)
      for (uint64_t run = me / t.parts; run < t.groups; run += t.abreast) {
        const uint64_t start = run * t.groupRows, end = start + t.groupRows < rows ? start + t.groupRows : rows;
        uint64_t row = start + me % t.parts;
        if (row < end && partial && partials < 2ull * t.teams + run * t.parts + me % t.parts + 1)
          partials = 2ull * t.teams + run * t.parts + me % t.parts + 1;
        for (; row < end; row += t.parts) {
          if (seen.c.gateRows > 1 && row / seen.c.gateRows != run && gate) die("a row of another group", rows, dim, gaterows);
          if (taken[row]++) die("a row twice", rows, dim, gaterows);
        }
      }
    for (uint64_t row = 0; row < rows; row++)
      if (!taken[row]) die("a row without a team", rows, dim, gaterows);
    if (partials * dim * 4 > bytes) die("partial rows outside of the workspace", rows, dim, gaterows);
    printf("%zu\n", bytes);
  }
  return 0;
}
