// embed_kernels.hip - rows of a table by token id, and the table's gradient.
//
// Lookup: out[t] = scale * table[ids[t] - first], zeros where the shard has no such row.  A
// gather of whole rows: memory bounds it, and every row is read and written in pieces of
// 16 bytes a lane.
//
// Gradient: G[v] = scale * sum of grad[t] over the tokens of row v.  A scatter with atomics
// would move fp32 read-modify-writes for every element and sum in an order that changes
// from run to run, so the tokens are sorted by row first (a stable radix sort of 32-bit
// keys, a few microseconds) and the sums become a stream over grad: a wavefront takes a
// chunk of consecutive sorted tokens and one slice of the columns, keeps the running sum
// in registers and writes a row when its last token is behind it.  A row whose tokens lie
// in several chunks leaves one fp32 partial sum in each, and a last kernel adds those in
// order: the work of one chunk is the same however often an id occurs.
//
// Compiled once per pair of types: -DFLAGCX_TABLE=<enum> -DFLAGCX_OUT=<enum>; the pair of
// fp32 and fp32 also holds what does not depend on types.
#include "launch.h"
#include "residual.h"
#include "residual_device.h"

namespace flagcx_amd {
namespace { // per unit: the same names stand for other types in the next one

#if FLAGCX_TABLE == 6
typedef h16 Tab;
#elif FLAGCX_TABLE == 7
typedef float Tab;
#else
typedef b16 Tab;
#endif
#if FLAGCX_OUT == 6
typedef h16 Out;
#elif FLAGCX_OUT == 7
typedef float Out;
#else
typedef b16 Out;
#endif
constexpr int kVec = 16 / (int)(sizeof(Tab) > sizeof(Out) ? sizeof(Tab) : sizeof(Out)); // 16 bytes of the wider type

// Row of the shard that token t names; `vocab` if the shard has none.
__device__ __forceinline__ uint64_t rowOf(const void *ids, bool wide, uint64_t t, int64_t first, uint64_t vocab) {
  const int64_t id = wide ? ((const int64_t *)ids)[t] : (int64_t)((const int32_t *)ids)[t];
  const uint64_t row = (uint64_t)id - (uint64_t)first;
  return id >= first && row < vocab ? row : vocab;
}

// ------------------------------------------------------------------ lookup

constexpr unsigned kMaxGrid = 1u << 20;

// blockDim = (lanes of a token, tokens of this workgroup)
template <int V>
__global__ void __launch_bounds__(256) embeddingKernel(EmbedCall p) {
  constexpr int U = 4; // vectors of a row in flight per lane
  const uint32_t lanes = blockDim.x;
  const uint64_t step = (uint64_t)gridDim.x * blockDim.y;
  for (uint64_t t = (uint64_t)blockIdx.x * blockDim.y + __builtin_amdgcn_readfirstlane(threadIdx.y); t < p.tokens; t += step) {
    const uint64_t row = rowOf(p.ids, p.wideIds != 0, t, p.first, p.vocab);
    const bool here = row < p.vocab;
    for (uint64_t at = 0; at < p.dim; at += (uint64_t)lanes * V * U) {
      const uint64_t left = p.dim - at;
      const uint32_t n = left < (uint64_t)lanes * V * U ? (uint32_t)left : lanes * V * U;
      const Row in((const Tab *)p.table + (here ? row * p.tableStride + at : 0), here ? n * (uint32_t)sizeof(Tab) : 0);
      const Row out((Out *)p.out + t * p.outStride + at, n * (uint32_t)sizeof(Out));
      Run<Tab, V> x[U];
#pragma unroll
      for (int u = 0; u < U; u++) x[u].load(in, u * lanes * V, threadIdx.x * V);
#pragma unroll
      for (int u = 0; u < U; u++) {
        Run<Out, V> y;
#pragma unroll
        for (int i = 0; i < V; i++) y.set(i, here ? p.scale * x[u].at(i) : 0.0f);
        y.template store<(V > 1 ? kAuxStream : kAuxPlain)>(out, u * lanes * V, threadIdx.x * V);
      }
    }
  }
}

template <int V>
int lookupFor(const EmbedCall &c, hipStream_t stream) {
  const uint64_t vecs = (c.dim + V - 1) / V;
  const uint32_t lanes = vecs <= 64 ? 64 : vecs <= 128 ? 128 : 256;
  const uint32_t per = 256 / lanes;
  const uint64_t groups = (c.tokens + per - 1) / per;
  embeddingKernel<V><<<dim3((unsigned)(groups < kMaxGrid ? groups : kMaxGrid)), dim3(lanes, per), 0, stream>>>(c);
  return (int)hipGetLastError();
}

} // namespace

// -------------------------------------------------------- gradient: layout

// Workspace: keys and tokens of the sorted order (twice: a pass reads one and writes the
// other), the passes' digit counts, and two partial rows per chunk.
struct GradPlan {
  uint32_t tokens, vocab;
  uint32_t passes, bits;  // digits of the keys 0 .. vocab
  uint32_t blocks, per;   // workgroups of a sorting pass and tokens each
  uint32_t chunk, chunks; // sorted tokens a wavefront sums
  uint32_t dimPad;        // floats between partial rows
  uint64_t bytes;
  uint64_t keyAt[2], tokAt[2], countAt, partAt;
};
GradPlan gradPlan(uint64_t tokens, uint64_t vocab, uint64_t dim);

int launchSort(const EmbedGradCall &c, const GradPlan &g, hipStream_t stream);

#if FLAGCX_TABLE == 7 && FLAGCX_OUT == 7
// ---------------------------------------------------------- gradient: sort

constexpr uint32_t kSortThreads = 256, kSortWaves = kSortThreads / 64;
constexpr uint32_t kMaxBits = 11, kMaxBins = 1u << kMaxBits;
constexpr uint32_t kMaxBlocks = 256;

GradPlan gradPlan(uint64_t tokens, uint64_t vocab, uint64_t dim) {
  GradPlan g{};
  g.tokens = (uint32_t)tokens;
  g.vocab = (uint32_t)vocab;
  uint32_t bits = 1;
  while (bits < 32 && (vocab >> bits) != 0) bits++;
  g.passes = (bits + kMaxBits - 1) / kMaxBits;
  g.bits = (bits + g.passes - 1) / g.passes;
  uint64_t blocks = (tokens + 2047) / 2048;
  if (blocks < 1) blocks = 1;
  if (blocks > kMaxBlocks) blocks = kMaxBlocks;
  g.per = (uint32_t)(((tokens + blocks - 1) / blocks + kSortThreads - 1) / kSortThreads * kSortThreads);
  if (g.per < kSortThreads) g.per = kSortThreads;
  g.blocks = (uint32_t)((tokens + g.per - 1) / g.per);
  if (g.blocks < 1) g.blocks = 1;
  // enough wavefronts to fill the chip before chunks grow
  const uint64_t slices = (dim + 511) / 512;
  g.chunk = 8;
  while (g.chunk < 32 && tokens * slices / g.chunk > 4096) g.chunk *= 2;
  g.chunks = (uint32_t)((tokens + g.chunk - 1) / g.chunk);
  g.dimPad = (uint32_t)((dim + 3) & ~3ull);
  uint64_t at = 0;
  auto take = [&at](uint64_t bytes) {
    const uint64_t here = at;
    at += (bytes + 255) & ~255ull;
    return here;
  };
  for (int i = 0; i < 2; i++) g.keyAt[i] = take(tokens * 4), g.tokAt[i] = take(tokens * 4);
  g.countAt = take((uint64_t)g.passes * g.blocks * (4u << g.bits));
  g.partAt = take((uint64_t)g.chunks * 2 * g.dimPad * 4);
  g.bytes = at;
  return g;
}

uint64_t embedGradWorkspace(uint64_t tokens, uint64_t vocab, uint64_t dim) { return gradPlan(tokens, vocab, dim).bytes; }

struct SortParams {
  const void *ids;
  int64_t first;
  int32_t wideIds;
  uint32_t tokens, vocab, per, blocks, bits, passes;
  uint32_t *counts;            // [pass][block][digit]
  const uint32_t *keyIn, *tokIn; // of passes after the first
  uint32_t *keyOut, *tokOut;
  uint32_t pass;
};

__device__ __forceinline__ uint32_t sortKey(const SortParams &p, uint32_t i) {
  return p.pass ? p.keyIn[i] : (uint32_t)rowOf(p.ids, p.wideIds != 0, i, p.first, p.vocab);
}

// Digit counts of the first pass; the later passes' counts start from zero.
__global__ void __launch_bounds__(kSortThreads) sortCountKernel(SortParams p) {
  __shared__ uint32_t hist[kMaxBins];
  const uint32_t bins = 1u << p.bits;
  for (uint32_t d = threadIdx.x; d < bins; d += kSortThreads) hist[d] = 0;
  __syncthreads();
  const uint32_t from = blockIdx.x * p.per, to = p.tokens - from < p.per ? p.tokens : from + p.per;
  for (uint32_t i = from + threadIdx.x; i < to; i += kSortThreads) atomicAdd(&hist[sortKey(p, i) & (bins - 1)], 1u);
  __syncthreads();
  for (uint32_t d = threadIdx.x; d < bins; d += kSortThreads) {
    p.counts[(uint64_t)blockIdx.x * bins + d] = hist[d];
    for (uint32_t q = 1; q < p.passes; q++) p.counts[((uint64_t)q * p.blocks + blockIdx.x) * bins + d] = 0;
  }
}

// One stable pass.  A workgroup's place for a digit: the digits before it, the same digit in
// the workgroups before it, then its own wavefronts in order, each of which takes its tokens
// 64 at a time and ranks equal digits by lane.
__global__ void __launch_bounds__(kSortThreads) sortPassKernel(SortParams p) {
  __shared__ uint32_t place[kSortWaves][kMaxBins];
  __shared__ uint32_t waveTotal[kSortWaves];
  const uint32_t bins = 1u << p.bits, shift = p.pass * p.bits;
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (uint32_t w = 0; w < kSortWaves; w++)
    for (uint32_t d = threadIdx.x; d < bins; d += kSortThreads) place[w][d] = 0;
  __syncthreads();
  const uint32_t from = blockIdx.x * p.per, to = p.tokens - from < p.per ? p.tokens : from + p.per;
  const uint32_t mine = p.per / kSortWaves; // tokens of a wavefront
  const uint32_t begin = from + wave * mine, end = begin + mine < to ? begin + mine : to;
  for (uint32_t i = begin + lane; i < end; i += 64) atomicAdd(&place[wave][(sortKey(p, i) >> shift) & (bins - 1)], 1u);
  __syncthreads();
  // this thread's run of digits: how many before this workgroup, how many in all
  const uint32_t run = bins > kSortThreads ? bins / kSortThreads : 1;
  constexpr uint32_t kMaxRun = kMaxBins / kSortThreads;
  uint32_t before[kMaxRun], total[kMaxRun], sum = 0;
  const uint32_t d0 = threadIdx.x * run;
#pragma unroll
  for (uint32_t r = 0; r < kMaxRun; r++) {
    before[r] = total[r] = 0;
    if (r < run && d0 + r < bins) {
      const uint32_t *c = p.counts + (uint64_t)p.pass * p.blocks * bins + d0 + r;
      for (uint32_t b = 0; b < p.blocks; b++) {
        const uint32_t n = c[(uint64_t)b * bins];
        if (b < blockIdx.x) before[r] += n;
        total[r] += n;
      }
      sum += total[r];
    }
  }
  uint32_t scan = sum; // inclusive over the wavefront's lanes
  for (uint32_t s = 1; s < 64; s *= 2) {
    const uint32_t o = __shfl_up(scan, s);
    if (lane >= s) scan += o;
  }
  if (lane == 63) waveTotal[wave] = scan;
  __syncthreads();
  uint32_t at = scan - sum;
  for (uint32_t w = 0; w < wave; w++) at += waveTotal[w];
#pragma unroll
  for (uint32_t r = 0; r < kMaxRun; r++) {
    if (r < run && d0 + r < bins) {
      uint32_t here = at + before[r];
      for (uint32_t w = 0; w < kSortWaves; w++) {
        const uint32_t n = place[w][d0 + r];
        place[w][d0 + r] = here;
        here += n;
      }
      at += total[r];
    }
  }
  __syncthreads();
  volatile uint32_t *next = place[wave]; // this wavefront's alone from here on
  for (uint32_t base = begin; base < end; base += 64) {
    const uint32_t i = base + lane;
    const bool live = i < end;
    const uint32_t key = live ? sortKey(p, i) : 0;
    const uint32_t token = live ? (p.pass ? p.tokIn[i] : i) : 0;
    const uint32_t digit = (key >> shift) & (bins - 1);
    uint64_t same = __ballot(live); // lanes with this lane's digit
    for (uint32_t b = 0; b < p.bits; b++) {
      const uint64_t set = __ballot((digit >> b) & 1u);
      same &= (digit >> b) & 1u ? set : ~set;
    }
    const uint32_t rank = (uint32_t)__popcll(same & ((1ull << lane) - 1ull));
    uint32_t to0 = 0;
    if (live) to0 = next[digit];
    __builtin_amdgcn_wave_barrier();
    if (live && rank == 0) next[digit] = to0 + (uint32_t)__popcll(same);
    __builtin_amdgcn_wave_barrier();
    if (live) {
      const uint32_t out = to0 + rank;
      p.keyOut[out] = key;
      p.tokOut[out] = token;
      if (p.pass + 1 < p.passes)
        atomicAdd(&p.counts[((uint64_t)(p.pass + 1) * p.blocks + out / p.per) * bins + ((key >> (shift + p.bits)) & (bins - 1))], 1u);
    }
  }
}

int launchSort(const EmbedGradCall &c, const GradPlan &g, hipStream_t stream) {
  char *ws = (char *)c.workspace;
  SortParams p{};
  p.ids = c.ids;
  p.first = c.first;
  p.wideIds = c.wideIds;
  p.tokens = g.tokens;
  p.vocab = g.vocab;
  p.per = g.per;
  p.blocks = g.blocks;
  p.bits = g.bits;
  p.passes = g.passes;
  p.counts = (uint32_t *)(ws + g.countAt);
  sortCountKernel<<<dim3(g.blocks), dim3(kSortThreads), 0, stream>>>(p);
  int e = (int)hipGetLastError();
  for (uint32_t q = 0; q < g.passes && !e; q++) {
    p.pass = q;
    p.keyIn = (const uint32_t *)(ws + g.keyAt[(q + 1) & 1]);
    p.tokIn = (const uint32_t *)(ws + g.tokAt[(q + 1) & 1]);
    p.keyOut = (uint32_t *)(ws + g.keyAt[q & 1]);
    p.tokOut = (uint32_t *)(ws + g.tokAt[q & 1]);
    sortPassKernel<<<dim3(g.blocks), dim3(kSortThreads), 0, stream>>>(p);
    e = (int)hipGetLastError();
  }
  return e;
}
#endif

// ---------------------------------------------------------- gradient: sums

namespace {

struct SumParams {
  const Out *grad;
  uint64_t gradStride;
  Tab *table;
  uint64_t tableStride;
  uint64_t dim;
  uint32_t slices; // workgroups that share a chunk
  uint32_t base;   // first chunk (or group of rows) of this launch
  uint32_t tokens, vocab, chunk, chunks, dimPad;
  float scale;
  int32_t accumulate;
  const uint32_t *key, *tok;
  float *part; // [chunk][2][dimPad]: a row that began before the chunk, a row that ends after it
};

template <int V>
__device__ __forceinline__ void writeRow(const SumParams &p, uint64_t row, uint64_t at, uint32_t n, uint32_t lane,
                                         const float (&sum)[V]) {
  const Row out(p.table + row * p.tableStride + at, n * (uint32_t)sizeof(Tab));
  Run<Tab, V> y;
  if (p.accumulate) {
    Run<Tab, V> old;
    old.load(out, 0, lane * V);
#pragma unroll
    for (int i = 0; i < V; i++) y.set(i, __builtin_fmaf(p.scale, sum[i], old.at(i)));
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) y.set(i, p.scale * sum[i]);
  }
  y.store(out, 0, lane * V);
}

template <int V>
__global__ void __launch_bounds__(256) gradSumKernel(SumParams p) {
  constexpr int B = 8; // rows of grad in flight
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t c = p.base + blockIdx.x / p.slices, slice = (blockIdx.x % p.slices) * (blockDim.x >> 6) + wave;
  const uint64_t at = (uint64_t)slice * 64 * V;
  if (at >= p.dim) return;
  const uint32_t n = p.dim - at < 64 * V ? (uint32_t)(p.dim - at) : 64 * V;
  const uint32_t from = c * p.chunk, count = p.tokens - from < p.chunk ? p.tokens - from : p.chunk;
  const uint32_t none = p.vocab;
  const uint32_t myKey = lane < count ? p.key[from + lane] : none;
  const uint32_t myTok = lane < count ? p.tok[from + lane] : 0;
  const uint32_t before = from ? p.key[from - 1] : ~0u, after = from + count < p.tokens ? p.key[from + count] : ~0u;
  float sum[V];
  uint32_t cur = __builtin_amdgcn_readlane(myKey, 0);
  bool began = before != cur; // the row's first token is in this chunk
#pragma unroll
  for (int i = 0; i < V; i++) sum[i] = -0.0f;
  auto finish = [&](bool ended) {
    if (began && ended) {
      writeRow<V>(p, cur, at, n, lane, sum);
    } else {
      const Row out(p.part + ((uint64_t)c * 2 + (began ? 1 : 0)) * p.dimPad + at, n * 4u);
      Run<float, V> y;
#pragma unroll
      for (int i = 0; i < V; i++) y.v[i] = sum[i];
      y.store(out, 0, lane * V);
    }
  };
  for (uint32_t i0 = 0; i0 < count; i0 += B) {
    Run<Out, V> x[B];
#pragma unroll
    for (int b = 0; b < B; b++) {
      const uint32_t k = __builtin_amdgcn_readlane(myKey, i0 + b), t = __builtin_amdgcn_readlane(myTok, i0 + b);
      const Row in(p.grad + (uint64_t)t * p.gradStride + at, k != none ? n * (uint32_t)sizeof(Out) : 0);
      x[b].template load<kAuxStream>(in, 0, lane * V);
    }
#pragma unroll
    for (int b = 0; b < B; b++) {
      const uint32_t k = __builtin_amdgcn_readlane(myKey, i0 + b);
      if (k != cur) {
        finish(true);
        cur = k;
        began = true;
#pragma unroll
        for (int i = 0; i < V; i++) sum[i] = -0.0f;
      }
      if (k == none) return; // behind the last token of the shard
#pragma unroll
      for (int i = 0; i < V; i++) sum[i] += x[b].at(i);
    }
  }
  finish(after != cur);
}

// Adds the partial sums of a row that spans chunks; a workgroup looks at one chunk in which such a row may begin.
constexpr uint32_t kJoinWaves = 4;
__global__ void __launch_bounds__(64 * kJoinWaves) gradJoinKernel(SumParams p) {
  __shared__ float part[kJoinWaves][64][4];
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t c = p.base + blockIdx.x / p.slices, slice = blockIdx.x % p.slices;
  if (c + 1 >= p.chunks) return;
  const uint32_t edge = (c + 1) * p.chunk, cur = p.key[edge - 1];
  if (cur == p.vocab || p.key[edge] != cur || (c && p.key[c * p.chunk - 1] == cur)) return;
  // the last chunk that begins with this row: a look at the next 64, then bisection
  uint32_t last = c + 1;
  {
    const uint32_t look = c + 1 + lane;
    const uint64_t same = __ballot(look < p.chunks && p.key[look < p.chunks ? look * p.chunk : 0] == cur);
    last = c + (same == ~0ull ? 64u : (uint32_t)__builtin_ctzll(~same));
    if (same == ~0ull) {
      uint32_t lo = last, hi = p.chunks - 1;
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        if (p.key[mid * p.chunk] == cur) lo = mid;
        else hi = mid - 1;
      }
      last = lo;
    }
  }
  const uint64_t at = (uint64_t)slice * 256;
  const uint32_t n = p.dim - at < 256 ? (uint32_t)(p.dim - at) : 256;
  const uint32_t padded = (n + 3) & ~3u;
  float sum[4] = {-0.0f, -0.0f, -0.0f, -0.0f};
  for (uint32_t i = c + wave; i <= last; i += kJoinWaves) {
    Run<float, 4> x;
    x.load(Row(p.part + ((uint64_t)i * 2 + (i == c ? 1 : 0)) * p.dimPad + at, padded * 4u), 0, lane * 4);
#pragma unroll
    for (int k = 0; k < 4; k++) sum[k] += x.v[k];
  }
#pragma unroll
  for (int k = 0; k < 4; k++) part[wave][lane][k] = sum[k];
  __syncthreads();
  if (wave) return;
  for (uint32_t w = 1; w < kJoinWaves; w++)
#pragma unroll
    for (int k = 0; k < 4; k++) sum[k] += part[w][lane][k];
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const float one[1] = {sum[k]};
    // element lane * 4 + k of the slice
    writeRow<1>(p, cur, at, n, lane * 4 + k, one);
  }
}

// Rows that no token names become zeros.  A workgroup takes 64 rows; one lane a row looks it up among the sorted keys.
constexpr uint32_t kZeroRows = 64;
template <int V>
__global__ void __launch_bounds__(256) gradZeroKernel(SumParams p) {
  __shared__ uint64_t hit;
  const uint64_t base = ((uint64_t)p.base + blockIdx.x) * kZeroRows;
  if (threadIdx.x < 64) {
    const uint64_t row = base + threadIdx.x;
    uint32_t lo = 0, hi = p.tokens; // first position whose key is not below row
    if (row < p.vocab) {
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (p.key[mid] < row) lo = mid + 1;
        else hi = mid;
      }
    }
    const uint64_t found = __ballot(row >= p.vocab || (lo < p.tokens && p.key[lo] == row));
    if (threadIdx.x == 0) hit = found;
  }
  __syncthreads();
  const uint64_t skip = hit;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Run<Tab, V> zero;
#pragma unroll
  for (int i = 0; i < V; i++) zero.set(i, 0.0f);
  for (uint32_t r = wave; r < kZeroRows; r += 4) {
    if ((skip >> r) & 1u) continue;
    for (uint64_t at = 0; at < p.dim; at += 64 * V * 4) {
      const uint32_t n = p.dim - at < 64 * V * 4 ? (uint32_t)(p.dim - at) : 64 * V * 4;
      const Row out(p.table + (base + r) * p.tableStride + at, n * (uint32_t)sizeof(Tab));
#pragma unroll
      for (int u = 0; u < 4; u++) zero.store(out, u * 64 * V, (threadIdx.x & 63u) * V);
    }
  }
}

// `parts` units of `each` workgroups in launches of at most kMaxGrid workgroups (or one unit).
template <typename K>
int inPieces(K kernel, SumParams p, uint32_t parts, uint32_t each, uint32_t threads, hipStream_t stream) {
  const uint32_t most = kMaxGrid / each > 0 ? kMaxGrid / each : 1;
  for (uint32_t base = 0; base < parts; base += most) {
    p.base = base;
    kernel<<<dim3((parts - base < most ? parts - base : most) * each), dim3(threads), 0, stream>>>(p);
    const int e = (int)hipGetLastError();
    if (e) return e;
  }
  return (int)hipSuccess;
}

template <int V>
int gradientFor(const EmbedGradCall &c, hipStream_t stream) {
  const GradPlan g = gradPlan(c.tokens, c.vocab, c.dim);
  char *ws = (char *)c.workspace;
  int e = (int)hipSuccess;
  if (c.tokens) e = launchSort(c, g, stream);
  if (e) return e;
  const uint32_t sorted = (g.passes - 1) & 1;
  SumParams p{};
  p.grad = (const Out *)c.grad;
  p.gradStride = c.gradStride;
  p.table = (Tab *)c.table;
  p.tableStride = c.tableStride;
  p.dim = c.dim;
  p.tokens = g.tokens;
  p.vocab = g.vocab;
  p.chunk = g.chunk;
  p.chunks = g.chunks;
  p.dimPad = g.dimPad;
  p.scale = c.scale;
  p.accumulate = c.accumulate;
  p.key = (const uint32_t *)(ws + g.keyAt[sorted]);
  p.tok = (const uint32_t *)(ws + g.tokAt[sorted]);
  p.part = (float *)(ws + g.partAt);
  if (!c.accumulate) e = inPieces(gradZeroKernel<V>, p, (uint32_t)((c.vocab + kZeroRows - 1) / kZeroRows), 1, 256, stream);
  if (e || !c.tokens) return e;
  const uint64_t waves = (c.dim + 64 * V - 1) / (64 * V);
  const uint32_t per = waves < 4 ? (uint32_t)waves : 4;
  p.slices = (uint32_t)((waves + per - 1) / per);
  e = inPieces(gradSumKernel<V>, p, g.chunks, p.slices, 64 * per, stream);
  if (e || g.chunks < 2) return e;
  p.slices = (uint32_t)((c.dim + 255) / 256);
  return inPieces(gradJoinKernel, p, g.chunks - 1, p.slices, 64 * kJoinWaves, stream);
}

} // namespace

#define FLAGCX_NAME2(a, x, y) a##_##x##_##y
#define FLAGCX_NAME(a, x, y) FLAGCX_NAME2(a, x, y)
int FLAGCX_NAME(launchEmbedding, FLAGCX_TABLE, FLAGCX_OUT)(const EmbedCall &c, hipStream_t stream) {
  return c.vec ? lookupFor<kVec>(c, stream) : lookupFor<1>(c, stream);
}
int FLAGCX_NAME(launchEmbeddingGrad, FLAGCX_TABLE, FLAGCX_OUT)(const EmbedGradCall &c, hipStream_t stream) {
  return c.vec ? gradientFor<kVec>(c, stream) : gradientFor<1>(c, stream);
}

} // namespace flagcx_amd
