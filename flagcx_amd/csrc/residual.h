// residual.h - what host_residual.cpp hands to the kernels of the residual stream after
// validation.  Strides are in elements.  Every launcher returns a hipError_t value.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace flagcx_amd {

constexpr int kNormMaxDim = 16384;
constexpr int kNormMaxRanks = 64;
constexpr uint32_t kNormNarrow = 256; // rows of up to so many elements: one wavefront, four elements a lane

struct NormCall {
  uint64_t rows;
  uint32_t dim;
  int32_t post, pre; // which norms
  int32_t weightF32; // weights are fp32 (else of the activations' type)
  float scale, eps, offset;
  const void *w1, *w2, *gate;
  uint64_t gateStride;
  uint64_t gateRows; // 0: one row of gates for all
  int32_t vec;       // every address and row stride is a multiple of 16 bytes, dim of 16 bytes' elements
};

struct NormForward {
  NormCall c;
  const void *src[kNormMaxRanks];
  int32_t k;
  uint64_t srcStride;
  const void *res;
  uint64_t resStride;
  void *resOut;
  uint64_t resOutStride;
  void *normOut;
  uint64_t normStride;
  void *sumOut;
  uint64_t sumStride;
};

// How the rows of a backward pass are shared out.  A run is the rows that share a row of gates, or
// all rows.  `abreast` runs are worked on at a time, each by `parts` teams, of which one takes every
// parts-th row; then the next ones.  Teams that run at the same time are on neighbouring rows: with
// stretches of rows a team they are a constant stride apart that aliases in the memory channels.
struct NormTeams {
  uint64_t groupRows, groups; // rows of a run (of the last one there may be fewer), runs
  uint32_t parts, abreast, teams;
};

struct NormBackward {
  NormCall c;
  const void *sum, *h, *dy, *dh; // dy or dh may be NULL
  uint64_t sumStride, hStride, dyStride, dhStride;
  void *ds, *dres; // or NULL
  uint64_t dsStride, dresStride;
  void *dw1, *dw2, *dgate; // or NULL
  uint64_t dgateStride;
  float *partial; // workspace: rows of dim floats, two for each team (dW1, dW2), then one for each part of a run (gates)
  NormTeams t;
};

// activations and residual stream, as flagcxDataType_t values
int launchNormForward(const NormForward &f, int act, int res, hipStream_t stream);
int launchNormBackward(const NormBackward &b, int act, int res, hipStream_t stream);

// The team that holds a row of `dim` elements: lanes (a multiple of 64) and elements a lane, 8 or 16 (of
// narrow rows, which are one wavefront's anyway, the launchers take 4).
struct TeamShape {
  uint32_t lanes;
  int elements;
};
inline TeamShape teamOf(uint32_t dim, int e) { return {((dim + (uint32_t)e - 1) / (uint32_t)e + 63u) & ~63u, e}; }
// Backward: two rows and the column sums of 8 elements fit the registers, of 16 they do not.
inline TeamShape backwardShape(uint32_t dim) { return teamOf(dim, dim <= 8192 ? 8 : 16); }
// Forward: wide rows of a long batch run better from fewer wavefronts (16384 x 6144: 275 us against 290; 8192 x 4096 not:
// 108 against 106; the widths between are not measured).  With few rows, lanes are what there is plenty of.
inline TeamShape forwardShape(uint32_t dim, uint64_t rows) {
  return teamOf(dim, dim <= 4096 || (dim <= 8192 && rows < 512) ? 8 : 16);
}
NormTeams normTeams(uint64_t rows, uint32_t dim, uint64_t gateRows);

struct EmbedCall {
  const void *table;
  uint64_t vocab, tableStride;
  uint32_t vec; // as above
  uint64_t dim;
  const void *ids;
  int32_t wideIds; // 64 bits
  uint64_t tokens;
  int64_t first;
  float scale;
  void *out;
  uint64_t outStride;
};
int launchEmbedding(const EmbedCall &c, int tabletype, int outtype, hipStream_t stream);

struct EmbedGradCall {
  const void *grad;
  uint64_t gradStride;
  uint32_t vec;
  uint64_t dim;
  const void *ids;
  int32_t wideIds;
  uint64_t tokens, vocab;
  int64_t first;
  float scale;
  void *table;
  uint64_t tableStride;
  int32_t accumulate;
  void *workspace;
};
uint64_t embedGradWorkspace(uint64_t tokens, uint64_t vocab, uint64_t dim);
int launchEmbeddingGrad(const EmbedGradCall &c, int outtype, int tabletype, hipStream_t stream);

} // namespace flagcx_amd
